"""The tail of a training step that learns from token log probabilities, as a program runs it: a pre-norm block's norm that
keeps its input in 8 bits, the output product, log probabilities and entropy, their gradient, the norm's output back from the 8
bits for the product's weight gradient, the norm's gradient.  Through both faces of the package, and over two column shards."""
import importlib

import pytest

import helpers  # noqa: F401  (paths)

pytestmark = pytest.mark.gpu

IGN = -100
EPS = 1e-6


def _values(q, scale, cols):
    import torch
    rows, nb = scale.shape
    step = ((scale.long() - 133 + 1023) << 52).view(torch.float64)
    return (q.double().view(rows, nb, 32) * step[..., None]).view(rows, nb * 32)[:, :cols]


def _run(face, x0, res, gamma, W, tok, g, h, sync):
    """One step; the products are torch's.  Everything the step leaves behind, by name."""
    import torch
    rows, cols = x0.shape
    vocab = W.shape[0]
    dev = x0.device
    o = {"z": torch.empty_like(x0), "x": torch.empty_like(res), "z8": torch.empty_like(x0), "dx0": torch.empty_like(x0),
         "dres": torch.empty_like(res), "dgamma": torch.empty_like(gamma)}
    hk = importlib.import_module("hotspa-ae_amd")
    o["q"], o["scale"] = hk.q8_empty(rows, cols, dev)
    for name in ("mu", "rs", "logprob", "entropy", "lse"):
        o[name] = torch.empty(rows, device=dev)
    o["top"], o["top_token"] = torch.empty((rows, 3), device=dev), torch.empty((rows, 3), dtype=torch.int64, device=dev)
    sync()
    face.add_ln_q8_fwd(x0, res, gamma, None, o["z"], o["x"], o["q"], o["scale"], o["mu"], o["rs"], EPS, True)
    sync()
    o["logits"] = o["z"].float() @ W.t()
    o["dlogits"] = torch.empty((rows, vocab), device=dev)
    sync()
    fwd, bwd = (face.token_logprob_fwd, face.token_logprob_bwd) if hasattr(face, "token_logprob_fwd") else \
        (face.token_logprob, face.token_logprob_gradient)
    fwd(o["logits"], tok, o["logprob"], o["entropy"], o["lse"], o["top"], o["top_token"], IGN)
    bwd(o["logits"], tok, o["lse"], o["entropy"], g, h, o["dlogits"], IGN)
    face.add_ln_q8_out(o["q"], o["scale"], o["mu"], o["rs"], gamma, None, o["z8"], True)
    sync()
    o["dW"] = o["dlogits"].t().contiguous() @ o["z8"].float()
    o["dz"] = (o["dlogits"] @ W).to(x0.dtype)
    sync()
    face.add_ln_q8_bwd(o["dz"], o["x"].to(o["dres"].dtype) * 0 + 0.5, o["q"], o["scale"], o["mu"], o["rs"], gamma, o["dx0"],
                       o["dres"], o["dgamma"], None, True)
    sync()
    return o


@pytest.mark.parametrize("dtype,rows,cols,vocab", [("bf16", 300, 512, 1003), ("fp32", 70, 257, 5000), ("bf16", 1500, 1024, 640)])
def test_step(hk, cuda, dtype, rows, cols, vocab):
    import torch
    ops = importlib.import_module("hotspa-ae_amd.hetu_ops")
    dt = {"bf16": torch.bfloat16, "fp32": torch.float32}[dtype]
    gen = torch.Generator(device=cuda).manual_seed(rows)

    def normal(*shape, std=1.0, t=dt):
        return (torch.randn(shape, generator=gen, device=cuda) * std).to(t)
    x0, res = normal(rows, cols), normal(rows, cols, std=2.0, t=torch.float32)
    gamma = (torch.rand(cols, generator=gen, device=cuda) + 0.5).to(dt)
    W = normal(vocab, cols, std=cols ** -0.5 * 2, t=torch.float32)
    tok = torch.randint(0, vocab, (rows,), generator=gen, device=cuda)
    tok[::9] = IGN
    g, h = normal(rows, t=torch.float32), normal(rows, std=0.1, t=torch.float32)
    a = _run(hk, x0, res, gamma, W, tok, g, h, torch.cuda.synchronize)
    b = _run(ops, x0, res, gamma, W, tok, g, h, lambda: (torch.cuda.synchronize(), ops.stream_sync()))
    for name in a:
        assert torch.equal(a[name], b[name]), name           # the two faces run the same kernels

    # against the definitions in 64 bits, step by step on what the step before left
    half = {"bf16": 2.0 ** -8, "fp32": 2.0 ** -24}[dtype]
    x = (x0.float() + res).double()
    rs = 1 / ((x * x).mean(1) + EPS).sqrt()
    z = gamma.double() * x * rs[:, None]
    assert bool(((a["z"].double() - z).abs() <= z.abs() * (half + 2.0 ** -17)).all())
    d = a["logits"].double()
    lp = torch.log_softmax(d, 1)
    p = lp.exp()
    H = -(p * lp).sum(1)
    live = tok != IGN
    want = lp.gather(1, tok.clamp(min=0)[:, None])[:, 0]
    # as in the log probabilities' own test: chains of fewer than 144 additions, values below 32
    assert bool(((a["logprob"].double() - want).abs()[live] <= 2.0 ** -16).all())
    assert bool(((a["entropy"].double() - H).abs()[live] <= 2.0 ** -12).all())
    assert bool((a["logprob"][~live] == 0).all()) and bool((a["entropy"][~live] == 0).all())
    one = torch.nn.functional.one_hot(tok.clamp(min=0), vocab).double()
    dl = g.double()[:, None] * (one - p) - h.double()[:, None] * p * (lp + H[:, None])
    dl[~live] = 0
    size = g.double().abs()[:, None] * (one + p) + h.double().abs()[:, None] * p * (lp.abs() + H[:, None])
    assert bool(((a["dlogits"].double() - dl).abs() <= 2.0 ** -14 * size + 2.0 ** -60).all())
    best = torch.sort(d, dim=1, descending=True, stable=True)[1][:, :3]
    assert torch.equal(a["top_token"][live], best[live]) and bool((a["top_token"][~live] == -1).all())
    x8 = _values(a["q"], a["scale"], cols)
    n8 = x8 * a["rs"].double()[:, None]
    z8 = gamma.double() * n8
    assert bool(((a["z8"].double() - z8).abs() <= z8.abs() * (half + 2.0 ** -21)).all())
    u = a["dz"].double() * gamma.double()
    dx = a["rs"].double()[:, None] * (u - n8 * (u * n8).mean(1, keepdim=True)) + 0.5
    err = 2.0 ** -16 * a["rs"].double()[:, None] * (u.abs() + n8.abs() * (u * n8).abs().mean(1, keepdim=True)) + 2.0 ** -22
    assert bool(((a["dres"].double() - dx).abs() <= err).all())
    assert bool(((a["dx0"].double() - dx).abs() <= err + dx.abs() * half).all())
    dg = (a["dz"].double() * n8)
    assert bool(((a["dgamma"].double() - dg.sum(0)).abs() <= 2.0 ** -17 * dg.abs().sum(0) + dg.sum(0).abs() * half).all())

    # what 8 bits cost: x8 is off by at most half a step, a step being at most 1/64 of the block's largest magnitude; the weight
    # gradient of the unrounded z differs by a product with that difference, bounded by the norms of its factors
    step = ((a["scale"].long() - 133 + 1023) << 52).view(torch.float64)
    off = (x8 - x).abs()
    assert bool((off <= step.repeat_interleave(32, 1)[:, :cols]).all())
    exact = a["dlogits"].double().t().contiguous() @ z
    gap = a["dlogits"].double().norm() * (a["z8"].double() - z).norm()
    assert float((a["dW"].double() - exact).norm()) <= float(gap) * (1 + 2.0 ** -10) + 2.0 ** -16 * float(exact.norm())


def test_step_over_two_shards(hk, cuda):
    """The same rows with the vocabulary over two column shards: what the shards' calls give is what the whole row's give."""
    import torch
    rows, vocab, cut = 300, 1003, 500
    gen = torch.Generator(device=cuda).manual_seed(4)
    logits = torch.randn((rows, vocab), generator=gen, device=cuda) * 3
    tok = torch.randint(0, vocab, (rows,), generator=gen, device=cuda)
    tok[::7] = IGN
    g, h = torch.randn(rows, generator=gen, device=cuda), torch.randn(rows, generator=gen, device=cuda)
    whole = [torch.empty(rows, device=cuda) for _ in range(3)]
    hk.token_logprob_fwd(logits, tok, *whole, None, None, IGN)
    ops = importlib.import_module("hotspa-ae_amd.hetu_ops")
    torch.cuda.synchronize()
    for face, sync in ((hk, lambda: None), (ops, ops.stream_sync)):
        stats = torch.empty((2, 4, rows), device=cuda)
        values, tokens = torch.empty((2, rows, 4), device=cuda), torch.empty((2, rows, 4), dtype=torch.int64, device=cuda)
        parts = [out.clone() for out in whole]
        value, token = torch.empty((rows, 4), device=cuda), torch.empty((rows, 4), dtype=torch.int64, device=cuda)
        torch.cuda.synchronize()
        for i, (first, last) in enumerate(((0, cut), (cut, vocab))):
            face.vocab_parallel_logprob_stats(logits[:, first:last], tok, stats[i], values[i], tokens[i], first, IGN)
        face.vocab_parallel_logprob_combine(stats, values, tokens, tok, IGN, *parts, value, token, vocab_size=vocab)
        sync()
        for a, b in zip(parts, whole):   # two fp32 computations, each within 2^-14 of values below 32 (see test_step)
            assert float((a - b).abs().max()) <= 2.0 ** -13
        dx = torch.empty_like(logits)
        ref = torch.empty_like(logits)
        bwd = face.token_logprob_bwd if face is hk else face.token_logprob_gradient
        torch.cuda.synchronize()
        for first, last in ((0, cut), (cut, vocab)):
            bwd(logits[:, first:last], tok, parts[2], parts[1], g, h, dx[:, first:last], IGN, vocab_start=first)
        sync()
        hk.token_logprob_bwd(logits, tok, parts[2], parts[1], g, h, ref, IGN)
        torch.cuda.synchronize()
        assert torch.equal(dx, ref)


def test_operator_layer_takes_any_layout(hk, cuda):
    """Views that the row kernels cannot read or write in place are gathered and laid back."""
    import torch
    ops = importlib.import_module("hotspa-ae_amd.hetu_ops")
    base = torch.randn((40, 3, 96), device=cuda)
    x = base.permute(1, 0, 2)                              # [3, 40, 96], rows not on one pitch
    dense = x.contiguous()
    tok = torch.randint(0, 96, (3, 40), device=cuda)
    for q_in in (x, dense):
        q, scale = hk.q8_empty(120, 96, cuda)
        torch.cuda.synchronize()
        ops.q8_pack(q_in, q, scale)
        ops.stream_sync()
        if q_in is x:
            kept = q.clone(), scale.clone()
    assert torch.equal(kept[0], q) and torch.equal(kept[1], scale)
    out = torch.zeros((40, 3, 96), device=cuda)
    lse, lp = torch.empty((3, 40), device=cuda), torch.empty((3, 40), device=cuda)
    grad = torch.ones((3, 40), device=cuda)
    torch.cuda.synchronize()
    ops.token_logprob(x, tok, lp, None, lse, None, None, IGN)
    ops.token_logprob_gradient(x, tok, lse, None, grad, None, out.permute(1, 0, 2), IGN)
    ops.stream_sync()
    ref = torch.empty_like(dense)
    hk.token_logprob_bwd(dense, tok, lse, None, grad, None, ref, IGN)
    torch.cuda.synchronize()
    assert torch.equal(out.permute(1, 0, 2), ref)
    z = torch.zeros((40, 3, 96), device=cuda)
    mu, rs = torch.empty(120, device=cuda), torch.empty(120, device=cuda)
    torch.cuda.synchronize()
    ops.add_ln_q8_fwd(x, None, None, None, z.permute(1, 0, 2), None, q, scale, mu, rs, EPS, False)
    ops.stream_sync()
    zz = torch.empty_like(dense)
    q2, scale2 = hk.q8_empty(120, 96, cuda)
    hk.add_ln_q8_fwd(dense, None, None, None, zz, None, q2, scale2, mu, rs, EPS, False)
    torch.cuda.synchronize()
    assert torch.equal(z.permute(1, 0, 2), zz) and torch.equal(q, q2)


def test_operator_layer_refusals(hk, cuda):
    import torch
    ops = importlib.import_module("hotspa-ae_amd.hetu_ops")
    x, tok, v = torch.zeros(4, 64, device=cuda), torch.zeros(4, dtype=torch.int64, device=cuda), torch.zeros(4, device=cuda)
    q, scale = hk.q8_empty(4, 64, cuda)
    for call in (lambda: ops.token_logprob(x, tok.int(), v, None, None, None, None, IGN),
                 lambda: ops.token_logprob(x, tok, v[:3], None, None, None, None, IGN),
                 lambda: ops.token_logprob(x, tok, v.half(), None, None, None, None, IGN),
                 lambda: ops.token_logprob(x, tok, v, None, None, torch.zeros(4, 2, device=cuda), None, IGN),
                 lambda: ops.token_logprob_gradient(x, tok, v, None, None, v, x, IGN),
                 lambda: ops.q8_pack(x, q[:3], scale), lambda: ops.q8_pack(x, q.to(torch.uint8), scale),
                 lambda: ops.add_ln_q8_fwd(x, None, v, None, x, None, q, scale, v, v, EPS, True),
                 lambda: ops.add_ln_q8_bwd(x, None, q, scale, v, v, None, x, None, None, torch.zeros(64, device=cuda), True)):
        with pytest.raises(ops.AssertionError_):
            call()
    with pytest.raises(ops.HetuError):
        ops.token_logprob(x.double(), tok, v, None, None, None, None, IGN)
    with pytest.raises(hk.HkError, match="dense"):
        hk.q8_pack(x, q.t(), scale)
    with pytest.raises(hk.HkError, match="float32"):
        hk.token_logprob_fwd(x, tok, v.half(), None, None, None, None, IGN)
    with pytest.raises(hk.HkError, match="one type"):
        hk.add_ln_q8_fwd(x, x, None, None, x, x.half(), q, scale, v, v, EPS, True)
    with pytest.raises(hk.HkError, match="shape"):
        hk.token_logprob_bwd(x, tok, v, None, v, None, x[:, :32], IGN)
    one = torch.zeros((), device=cuda)
    for call in (lambda: hk.token_logprob_fwd(one, tok, v, None, None, None, None, IGN),
                 lambda: hk.token_logprob_bwd(one, tok, v, None, v, None, one, IGN),
                 lambda: hk.vocab_parallel_logprob_stats(one, tok, torch.zeros(4, 1, device=cuda), None, None, 0, IGN),
                 lambda: hk.q8_pack(one, q, scale), lambda: hk.q8_unpack(q, scale, one),
                 lambda: hk.add_ln_q8_fwd(one, None, None, None, one, None, q, scale, v, v, EPS, True),
                 lambda: hk.add_ln_q8_out(q, scale, v, v, None, None, one, True)):
        with pytest.raises(hk.HkError, match="scalar"):
            call()
    with pytest.raises(hk.HkError, match="unit-stride"):
        hk.token_logprob_fwd(torch.zeros(64, 4, device=cuda).t(), tok, v, None, None, None, None, IGN)
