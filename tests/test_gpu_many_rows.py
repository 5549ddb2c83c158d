"""Log probabilities and 8-bit checkpoints of more rows than one launch's threads can be counted in 32 bits, and of rows whose
offsets pass them: what two calls on the parts give."""
import pytest

import helpers  # noqa: F401  (paths)

pytestmark = pytest.mark.gpu

IGN = -100


def _room(torch, gib):
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip("needs %d GiB of GPU memory" % gib)


@pytest.mark.parametrize("top", [0, 2])
def test_token_logprob_of_many_rows(hk, cuda, top):
    import torch
    _room(torch, 8)
    rows, cut = (1 << 25) + 37, 1 << 25
    gen = torch.Generator(device=cuda).manual_seed(1)
    x = torch.randn((rows, 3), generator=gen, device=cuda).to(torch.bfloat16)
    tok = torch.randint(0, 3, (rows,), generator=gen, device=cuda)
    tok[5], tok[rows - 5] = IGN, IGN

    def run(lo, hi):
        n = hi - lo
        o = [torch.full((n,), 9.0, device=cuda) for _ in range(3)]
        o += [torch.full((n, top), 9.0, device=cuda), torch.full((n, top), 9, dtype=torch.int64, device=cuda)] if top else [None, None]
        hk.token_logprob_fwd(x[lo:hi], tok[lo:hi], *o, IGN)
        dx = torch.full((n, 3), 9.0, dtype=torch.bfloat16, device=cuda)
        hk.token_logprob_bwd(x[lo:hi], tok[lo:hi], o[2], o[1], o[0], o[1], dx, IGN)
        stats = torch.full((1, 4, n), 9.0, device=cuda)
        value, token = (torch.empty((1, n, top), device=cuda), torch.empty((1, n, top), dtype=torch.int64, device=cuda)) \
            if top else (None, None)
        hk.vocab_parallel_logprob_stats(x[lo:hi], tok[lo:hi], stats[0], value[0] if top else None, token[0] if top else None, 0, IGN)
        c = [torch.full_like(t, 7) if t is not None else None for t in o]
        hk.vocab_parallel_logprob_combine(stats, value, token, tok[lo:hi], IGN, *c, vocab_size=3)
        return [t for t in o + [dx, stats.view(4, n).t()] + c if t is not None]

    whole = run(0, rows)
    for lo, hi in ((0, 1000), (cut - 1000, cut), (cut // 2 - 500, cut // 2 + 500), (cut, rows)):
        for a, b in zip(whole, run(lo, hi)):
            assert torch.equal(a[lo:hi], b), (lo, hi)
    for t in whole[:2]:
        assert bool((t != 9).all())          # every row was written


def test_norm_of_many_rows(hk, cuda):
    import torch
    _room(torch, 40)
    rows, cut, cols = (1 << 28) + 50, 1 << 28, 2
    x = torch.empty((rows, cols), dtype=torch.bfloat16, device=cuda).uniform_(-2, 2)
    res = torch.empty_like(x).uniform_(-2, 2)

    def run(lo, hi):
        n = hi - lo
        q, scale = hk.q8_empty(n, cols, cuda)
        mu, rs = torch.full((n,), 9.0, device=cuda), torch.full((n,), 9.0, device=cuda)
        z, out = torch.empty_like(x[lo:hi]), torch.empty_like(x[lo:hi])
        hk.add_ln_q8_fwd(x[lo:hi], res[lo:hi], None, None, z, out, q, scale, mu, rs, 1e-5, False)
        z8 = torch.empty_like(z)
        hk.add_ln_q8_out(q, scale, mu, rs, None, None, z8, False)
        dx = torch.empty_like(z)
        hk.add_ln_q8_bwd(z, None, q, scale, mu, rs, None, dx, None, None, None, False)
        return q, scale, mu, rs, z, out, z8, dx

    whole = run(0, rows)
    for lo, hi in ((0, 1000), (cut - 1000, cut), (cut // 2 - 500, cut // 2 + 500), (cut, rows)):
        for a, b in zip(whole, run(lo, hi)):
            assert torch.equal(a[lo:hi], b), (lo, hi)
    assert bool((whole[2] != 9).all())


@pytest.mark.parametrize("dtype,rows,past", [("bf16", 1, 77), ("fp32", 2, 40)])
def test_rows_that_are_packed_in_pieces(hk, cuda, dtype, rows, past):
    import torch
    _room(torch, 16)
    dt = {"bf16": torch.bfloat16, "fp32": torch.float32}[dtype]
    run = 1 << 28
    cols = (run if rows == 2 else 4 * run) + past        # the offsets of 4 runs pass 31 bits
    x = torch.empty((rows, cols), dtype=dt, device=cuda).uniform_(-3, 3)
    q, scale = hk.q8_empty(rows, cols, cuda)
    hk.q8_pack(x, q, scale)
    out = torch.zeros_like(x)
    hk.q8_unpack(q, scale, out)
    for r in range(rows):
        for c in range(0, cols, run):
            n = min(run, cols - c)
            wide = 1 << 14 if n == run else n            # as rows of other lengths
            part = x[r, c:c + n].view(-1, wide)
            q2, scale2 = hk.q8_empty(n // wide, wide, cuda)
            hk.q8_pack(part, q2, scale2)
            back = torch.empty_like(part)
            hk.q8_unpack(q2, scale2, back)
            nb = -(-n // 32)
            assert torch.equal(q[r, c:c + nb * 32], q2.view(-1)) and torch.equal(scale[r, c // 32:c // 32 + nb], scale2.view(-1))
            assert torch.equal(out[r, c:c + n], back.view(-1))
