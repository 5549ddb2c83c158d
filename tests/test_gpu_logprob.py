"""GPU parity of the token log probabilities, their entropy and alternatives, their gradient and their vocabulary-parallel
form (hk_token_logprob_*, hk_vocab_parallel_logprob_*) against the definitions in 64 bits."""
import math

import pytest

import helpers

pytestmark = pytest.mark.gpu

IGN = -100
TYPES = ("fp32", "bf16", "fp16")


def _dt(name):
    import torch
    return {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}[name]


def _make(rows, cols, dtype, seed=1, std=2.5, ignored=0.2, cuda="cuda"):
    import torch
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = (torch.randn((rows, cols), generator=g, device=cuda) * std - 3).to(_dt(dtype))
    tok = torch.randint(0, cols, (rows,), generator=g, device=cuda)
    tok[torch.rand(rows, generator=g, device=cuda) < ignored] = IGN
    tok[0] = cols - 1
    return x, tok


def _reference(x, tok, top):
    """logprob, entropy, lse, mean distance to the maximum, values and tokens of the alternatives, in 64 bits."""
    import torch
    d = x.double()
    rows, cols = d.shape
    m = d.amax(1, keepdim=True)
    e = torch.exp(d - m)
    s = e.sum(1)
    lse = m[:, 0] + torch.log(s)
    far = torch.where(e > 0, d - m, torch.zeros_like(d))
    dist = -(e * far).sum(1) / s
    entropy = torch.log(s) + dist
    inside = (tok >= 0) & (tok < cols)
    lp = d.gather(1, tok.clamp(0, cols - 1)[:, None])[:, 0] - lse
    lp = torch.where(inside, lp, torch.full_like(lp, math.nan))
    k = min(top, cols)
    v, i = torch.sort(d, dim=1, descending=True, stable=True)
    values = torch.full((rows, top), -math.inf, dtype=torch.float64, device=x.device)
    tokens = torch.full((rows, top), -1, dtype=torch.int64, device=x.device)
    values[:, :k] = v[:, :k] - lse[:, None]
    tokens[:, :k] = torch.where(v[:, :k] == -math.inf, torch.full_like(i[:, :k], -1), i[:, :k])
    ign = tok == IGN
    for t in (lp, entropy, lse):
        t[ign] = 0
    values[ign], tokens[ign] = -math.inf, -1
    return lp, entropy, lse, dist, values, tokens


def _run(hk, x, tok, top, workspace=None):
    import torch
    rows = x.shape[0]
    out = [torch.full((rows,), 7.0, device=x.device) for _ in range(3)]
    value = torch.full((rows, top), 7.0, device=x.device) if top else None
    token = torch.full((rows, top), 77, dtype=torch.int64, device=x.device) if top else None
    hk.token_logprob_fwd(x, tok, *out, value, token, IGN, workspace=workspace)
    torch.cuda.synchronize()
    return out + [value, token]


def _check(got, want, what=""):
    """fp32 arithmetic on exact inputs.  log S: a term exp(d), d = x - m <= 0, carries the roundings of d, of d log2(e) and of
    the exponential, 2^-24 (2 |d| + 2) of itself, which sums to 2^-23 (dist + 1) of S, dist = the mean of |d| under p; a chain of
    up to 128 additions and some 16 merges adds at most 144 * 2^-24 < 2^-16.8 of S.  The moment W likewise, of |W| = dist S.
    Final roundings: 2^-23 of each of the terms m, log S, dist."""
    lp, entropy, lse, dist, values, tokens = want
    import torch
    rel = 2.0 ** -16.8 + 2.0 ** -23 * (dist + 1)
    live = torch.isfinite(lse)
    size = lse.abs() + entropy.abs() + dist + 1
    e_lse = rel + 2.0 ** -22 * size
    for name, a, b, bound in (("lse", got[2], lse, e_lse),
                              ("logprob", got[0], lp, e_lse + 2.0 ** -23 * lp.abs().nan_to_num()),
                              ("entropy", got[1], entropy, rel * (1 + 2 * dist) + 2.0 ** -22 * size)):
        a = a.double()
        b = torch.where(b.abs() < 2.0 ** 128, b, b.float().double())   # past fp32's range a value is an infinity
        same = torch.isfinite(b) == torch.isfinite(a)
        assert bool(same.all()), (what, name, a[~same][:4], b[~same][:4])
        fin = torch.isfinite(b) & live
        assert bool(((a - b).abs() <= bound)[fin].all()), (what, name, float(((a - b).abs() / bound)[fin].max()))
    if tokens.shape[1]:
        assert torch.equal(got[4], tokens), (what, (got[4] != tokens).nonzero()[:4], got[4][:2], tokens[:2])
        a, b = got[3].double(), values
        b = torch.where(b.abs() < 2.0 ** 128, b, b.float().double())
        fin = torch.isfinite(b)
        assert bool((torch.isfinite(a) == fin).all()), what
        bound = (e_lse[:, None] + 2.0 ** -23 * b.abs()).expand_as(b)
        assert bool(((a - b).abs() <= bound)[fin].all()), what


SHAPES = [(1, 1), (1, 2), (3, 7), (5, 8), (9, 64), (2, 65), (33, 1000), (7, 4099), (700, 1003), (600, 513), (2, 50257),
          (1, 131080), (64, 32000), (515, 8192), (1, 300001)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("top", [0, 5])
def test_forward(hk, cuda, dtype, shape, top):
    x, tok = _make(*shape, dtype)
    _check(_run(hk, x, tok, top), _reference(x, tok, top), (dtype, shape))


@pytest.mark.parametrize("top", [1, 2, 20, 31, 32])
@pytest.mark.parametrize("shape", [(3, 7), (4, 33), (9, 1024), (600, 2000), (1, 50257), (40, 30011)])
def test_number_of_alternatives(hk, cuda, top, shape):
    x, tok = _make(*shape, "bf16", seed=3, ignored=0.1)
    _check(_run(hk, x, tok, top), _reference(x, tok, top), (shape, top))


@pytest.mark.parametrize("dtype", TYPES)
def test_equal_logits_go_to_the_lowest_token(hk, cuda, dtype):
    """Constant rows, rows of few values, both zeros, and more equal ones than the list of candidates holds."""
    import torch
    for rows, cols in ((4, 40), (3, 5000), (2, 70001), (600, 1500)):
        g = torch.Generator(device=cuda).manual_seed(cols)
        x = torch.randint(0, 3, (rows, cols), generator=g, device=cuda).to(_dt(dtype)) * 0.5
        x[0] = 1.25
        x[1] = torch.where(torch.rand(cols, generator=g, device=cuda) < 0.5, 0.0, -0.0).to(x.dtype)
        tok = torch.zeros(rows, dtype=torch.int64, device=cuda)
        _check(_run(hk, x, tok, 20), _reference(x, tok, 20), (dtype, rows, cols))


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_logits(hk, cuda, dtype):
    """-inf, the type's lowest value and rows that have little or nothing else."""
    import torch
    low = torch.finfo(_dt(dtype)).min
    for cols in (6, 1003, 40000):
        x, tok = _make(8, cols, dtype, seed=cols, ignored=0.0)
        x[0, ::2] = -math.inf
        x[1, 1:] = -math.inf               # one left
        x[2] = -math.inf                   # none
        x[3, ::3] = low
        x[4] = low                         # all equal, at the end of the range
        x[5] = torch.finfo(x.dtype).max
        x[6, 2:] = -math.inf
        x[6, 0] = low
        x[6, 1] = torch.finfo(x.dtype).max
        tok[:] = 0
        tok[7] = cols                      # outside
        want = _reference(x, tok, 4)
        lp, entropy, lse, dist, values, tokens = want
        lp[2] = entropy[2] = math.nan
        dist[2] = 0
        values[2], tokens[2] = math.nan, -1
        got = _run(hk, x, tok, 4)
        assert math.isnan(float(got[0][2])) and math.isnan(float(got[1][2])) and float(got[2][2]) == -math.inf
        assert bool(torch.isnan(got[3][2]).all()) and math.isnan(float(got[0][7]))
        _check(got, want, (dtype, cols))


def test_rows_without_a_distribution(hk, cuda):
    import torch
    for cols in (9, 3001, 60000):
        x, tok = _make(4, cols, "fp32", ignored=0.0)
        x[1, cols // 2] = math.nan
        x[2, cols - 1] = math.inf
        x[3, 0] = -math.nan
        got = _run(hk, x, tok, 3)
        want = _reference(x[:1], tok[:1], 3)
        _check([g[:1] for g in got], want)
        for r in (1, 2, 3):
            assert all(math.isnan(float(got[i][r])) for i in (0, 1)) and bool(torch.isnan(got[3][r]).all())
            assert got[4][r].tolist() == [-1] * 3


@pytest.mark.parametrize("dtype", TYPES)
def test_pitch_and_neighbours(hk, cuda, dtype):
    """Rows of a wider array at any boundary; nothing beside the outputs is written; some outputs left out."""
    import torch
    rows, cols = 37, 2051
    wide = torch.randn((rows, cols + 29), device=cuda).to(_dt(dtype))
    for first in (0, 1, 3, 8):
        x = wide[:, first:first + cols]
        tok = torch.randint(0, cols, (rows,), device=cuda)
        want = _reference(x.contiguous(), tok, 6)
        _check(_run(hk, x, tok, 6), want)
        buf = torch.full((rows + 8,), 5.0, device=cuda)
        hk.token_logprob_fwd(x, tok, buf[4:4 + rows], None, None, None, None, IGN)
        assert torch.equal(buf[:4], torch.full((4,), 5.0, device=cuda)) and torch.equal(buf[4 + rows:], buf[:4])
        out = torch.full((rows, cols + 8), 3.0, device=cuda).to(x.dtype)
        grad = torch.randn(rows, device=cuda)
        lse = want[2].float()
        hk.token_logprob_bwd(x, tok, lse, None, grad, None, out[:, 4:4 + cols], IGN)
        assert bool((out[:, :4] == 3).all()) and bool((out[:, 4 + cols:] == 3).all())
        ref = torch.empty_like(x.contiguous())
        hk.token_logprob_bwd(x.contiguous(), tok, lse, None, grad, None, ref, IGN)
        assert torch.equal(out[:, 4:4 + cols], ref)


def test_rows_far_apart(hk, cuda):
    """Offsets past 2^31 elements."""
    import torch
    pitch, cols = (1 << 30) + 8, 5003
    base = torch.empty(pitch * 2 + cols, dtype=torch.bfloat16, device=cuda)
    x = base.as_strided((3, cols), (pitch, 1))
    x.copy_(torch.randn((3, cols), device=cuda))
    tok = torch.tensor([1, 2, 3], device=cuda)
    want = _reference(x.contiguous(), tok, 3)
    _check(_run(hk, x, tok, 3), want)
    dense = x.contiguous()
    grad = torch.ones(3, device=cuda)
    ref = torch.empty_like(dense)
    hk.token_logprob_bwd(dense, tok, want[2].float(), None, grad, None, ref, IGN)
    hk.token_logprob_bwd(x, tok, want[2].float(), None, grad, None, x, IGN)
    assert torch.equal(x.contiguous(), ref)


# ------------------------------- gradient ----------------------------------
def _gradient(x, tok, g, h, start=0, lse=None, entropy=None):
    import torch
    d = x.double()
    lse = torch.logsumexp(d, 1) if lse is None else lse.double()
    lp = d - lse[:, None]
    p = torch.exp(lp)
    one = (torch.arange(x.shape[1], device=x.device)[None] + start == tok[:, None]).double()
    out = g.double()[:, None] * (one - p)
    terms = g.double().abs()[:, None] * (one + p)
    plp = torch.where(p > 0, p * lp, torch.zeros_like(p))
    if h is not None:
        H = -plp.sum(1) if entropy is None else entropy.double()
        out = out - h.double()[:, None] * (plp + p * H[:, None])
        terms = terms + h.double().abs()[:, None] * (plp.abs() + p * H.abs()[:, None])
    ign = (tok == IGN)[:, None]
    return out.masked_fill(ign, 0), terms.masked_fill(ign, 0), lse, lp


def _check_gradient(got, want, terms, lse, lp, dtype, what=""):
    """lse is handed over rounded to fp32 and x - lse and its product with log2(e) are rounded: 2^-23 (|lse| + |x - lse|) in the
    exponent, the exponential 2^-23, five more operations 2^-24 of the terms each, and the storage type's rounding; fp16 has
    magnitudes below 2^-14 in steps of 2^-24."""
    import torch
    lp = lp.nan_to_num(neginf=0.0)
    rel = 2.0 ** -22 * (lse.abs()[:, None] + lp.abs()) + 2.0 ** -20
    bound = terms * rel + want.abs() * {"fp32": 0.0, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}[dtype]
    bound = bound + (2.0 ** -24 if dtype == "fp16" else 2.0 ** -126)
    bad = (got.double() - want).abs() > bound
    assert not bool(bad.any()), (what, bad.nonzero()[:4], float(((got.double() - want).abs() / bound).max()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (9, 64), (33, 1000), (7, 4099), (700, 1003), (5, 50257), (2, 131080)])
@pytest.mark.parametrize("entropy", [False, True])
def test_gradient(hk, cuda, dtype, shape, entropy):
    import torch
    x, tok = _make(*shape, dtype, seed=5)
    rows = shape[0]
    lse, ent = torch.empty(rows, device=cuda), torch.empty(rows, device=cuda)
    hk.token_logprob_fwd(x, tok, None, ent, lse, None, None, IGN)
    g, h = torch.randn(rows, device=cuda), torch.randn(rows, device=cuda) * 0.1
    out = torch.full_like(x, 9.0)
    hk.token_logprob_bwd(x, tok, lse, ent if entropy else None, g, h if entropy else None, out, IGN)
    want, terms, _, lp = _gradient(x, tok, g, h if entropy else None, lse=torch.where(tok == IGN, 0, lse), entropy=ent)
    live = tok != IGN
    _check_gradient(out[live], want[live], terms[live], lse[live], lp[live], dtype, (dtype, shape))
    assert bool((out[~live] == 0).all())
    only = torch.empty_like(x)
    if entropy:
        hk.token_logprob_bwd(x, tok, lse, ent, None, h, only, IGN)
        want, terms, _, lp = _gradient(x, tok, torch.zeros_like(g), h, lse=lse, entropy=ent)
        _check_gradient(only[live], want[live], terms[live], lse[live], lp[live], dtype)
    again = x.clone()
    hk.token_logprob_bwd(again, tok, lse, ent if entropy else None, g, h if entropy else None, again, IGN)   # in place
    assert torch.equal(again, out)


@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_of_masked_logits(hk, cuda, dtype):
    import torch
    x, tok = _make(6, 1500, dtype, seed=8, ignored=0.0)
    x[:, 100:900] = -math.inf
    x[1, 1:] = -math.inf
    x[2, 1:] = torch.finfo(x.dtype).min
    tok[:] = 0
    tok[3] = 200                       # a masked token
    tok[4] = 5000                      # a token that the row does not have
    rows = 6
    ent, lse = torch.empty(rows, device=cuda), torch.empty(rows, device=cuda)
    hk.token_logprob_fwd(x, tok, None, ent, lse, None, None, IGN)
    g, h = torch.randn(rows, device=cuda), torch.randn(rows, device=cuda) * 1e6
    out = torch.empty_like(x)
    hk.token_logprob_bwd(x, tok, lse, ent, g, h, out, IGN)
    want, terms, lse64, lp = _gradient(x, tok, g, h, lse=lse, entropy=ent)
    assert bool(torch.isfinite(out.float()).all()) or dtype == "fp16"
    fin = torch.isfinite(out.float())
    _check_gradient(torch.where(fin, out, torch.zeros_like(out)), torch.where(fin, want, torch.zeros_like(want)), terms, lse, lp,
                    dtype)


def test_gradient_against_differences(hk, cuda):
    """Central differences of the forward pass.  Third derivatives of both functions are below 8 here (they are sums of
    products of probabilities and log probabilities, |log p| < 8): the step 2^-5 leaves 2^-10 * 8 / 6; the values' own error,
    2^-19 of sizes below 8, divided by the step, 2^-11."""
    import torch
    rows, cols, step = 3, 11, 2.0 ** -5
    x = torch.randn((rows, cols), device=cuda)
    tok = torch.tensor([0, 10, 4], device=cuda)
    lse, ent = torch.empty(rows, device=cuda), torch.empty(rows, device=cuda)
    hk.token_logprob_fwd(x, tok, None, ent, lse, None, None, IGN)
    for which in (0, 1):
        one = torch.ones(rows, device=cuda)
        grad = torch.empty_like(x)
        hk.token_logprob_bwd(x, tok, lse, ent, one if which == 0 else None, one if which else None, grad, IGN)
        for c in range(cols):
            ends = []
            for sign in (1, -1):
                y = x.clone()
                y[:, c] += sign * step
                ends.append(_run(hk, y, tok, 0)[which])
            diff = (ends[0] - ends[1]) / (2 * step)
            assert bool(((diff - grad[:, c]).abs() <= 2.0 ** -9 + 2.0 ** -10).all()), (which, c, diff, grad[:, c])


# ------------------------------- shards ------------------------------------
def _shards(hk, x, tok, widths, top, order=None):
    import torch
    rows, n = x.shape[0], len(widths)
    stats = torch.full((n, 4, rows), 7.0, device=x.device)
    values = torch.full((n, rows, top), 7.0, device=x.device) if top else None
    tokens = torch.full((n, rows, top), 77, dtype=torch.int64, device=x.device) if top else None
    starts = [sum(widths[:i]) for i in range(n)]
    for place, i in enumerate(order or range(n)):
        part = x[:, starts[i]:starts[i] + widths[i]]
        hk.vocab_parallel_logprob_stats(part, tok, stats[place], values[place] if top else None, tokens[place] if top else None,
                                        starts[i], IGN)
    out = [torch.full((rows,), 7.0, device=x.device) for _ in range(3)]
    value = torch.full((rows, top), 7.0, device=x.device) if top else None
    token = torch.full((rows, top), 77, dtype=torch.int64, device=x.device) if top else None
    hk.vocab_parallel_logprob_combine(stats, values, tokens, tok, IGN, *out, value, token, vocab_size=x.shape[1])
    torch.cuda.synchronize()
    return out + [value, token]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,widths", [(1, [5]), (3, [1, 1]), (5, [3, 40, 7]), (600, [500, 503]), (9, [4000] * 8),
                                         (2, [12565] * 4), (70, [64] * 64), (1, [30000, 1])])
@pytest.mark.parametrize("top", [0, 6])
def test_shards(hk, cuda, dtype, rows, widths, top):
    x, tok = _make(rows, sum(widths), dtype, seed=11)
    want = _reference(x, tok, top)
    _check(_shards(hk, x, tok, widths, top), want, (dtype, rows, widths))
    _check(_shards(hk, x, tok, widths, top, list(range(len(widths)))[::-1]), want)
    # the gradient of a shard is the columns of the whole row's
    import torch
    lse, ent = want[2].float(), want[1].float()
    g, h = torch.randn(rows, device=cuda), torch.randn(rows, device=cuda)
    whole = torch.empty_like(x)
    hk.token_logprob_bwd(x, tok, lse, ent, g, h, whole, IGN)
    start = 0
    for w in widths:
        part = torch.empty((rows, w), dtype=x.dtype, device=cuda)
        hk.token_logprob_bwd(x[:, start:start + w], tok, lse, ent, g, h, part, IGN, vocab_start=start)
        assert torch.equal(part, whole[:, start:start + w])
        start += w


def test_shards_with_equal_and_masked_logits(hk, cuda):
    import torch
    x = torch.zeros((7, 600), device=cuda)
    x[1, 200:400] = -math.inf              # a shard without a token
    x[2] = -math.inf
    x[3, 250] = math.nan
    x[4, 300:] = 1.0
    tok = torch.tensor([599, 0, 5, 5, 5, IGN, 600], device=cuda)
    want = _reference(x, tok, 5)
    lp, entropy, lse, dist, values, tokens = want
    for r in (2, 3):
        lp[r] = entropy[r] = math.nan
        dist[r] = 0
        values[r], tokens[r] = math.nan, -1
    lse[2], lse[3] = -math.inf, math.nan
    got = _shards(hk, x, tok, [200] * 3, 5)
    assert bool(torch.isnan(got[3][2:4]).all()) and math.isnan(float(got[0][6]))
    _check(got, want)


# ------------------------------- how it is called ---------------------------
def test_replayed_graph_and_other_stream(hk, cuda):
    """Captured on a stream of its own, replayed with new inputs between eager calls; two graphs share a workspace."""
    import torch
    shapes = [(3, 40001), (600, 2003)]
    state = []
    need = max(hk.token_logprob_workspace_bytes(8, r, c, 5) for r, c in shapes)
    ws = torch.empty(need // 4 + 2, device=cuda)
    side = torch.cuda.Stream()
    for r, c in shapes:
        x, tok = _make(r, c, "bf16", seed=c)
        out = [torch.empty(r, device=cuda) for _ in range(3)]
        value, token = torch.empty((r, 5), device=cuda), torch.empty((r, 5), dtype=torch.int64, device=cuda)
        dx = torch.empty_like(x)
        g = torch.randn(r, device=cuda)

        def call(x=x, tok=tok, out=out, value=value, token=token, dx=dx, g=g):
            hk.token_logprob_fwd(x, tok, *out, value, token, IGN, workspace=ws)
            hk.token_logprob_bwd(x, tok, out[2], out[1], g, g, dx, IGN)
        with torch.cuda.stream(side):
            call()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call()
        state.append((graph, call, x, tok, out, value, token, dx))
    for turn in range(3):
        for graph, call, x, tok, out, value, token, dx in state:
            x.copy_((torch.randn(x.shape, device=cuda) * (turn + 1)).to(x.dtype))
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in (*out, value, token, dx)]
            call()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, (*out, value, token, dx)))
            _check(got[:5], _reference(x, tok, 5), turn)


def test_results_repeat(hk, cuda):
    import torch
    x, tok = _make(200, 30000, "bf16")
    first = _run(hk, x, tok, 20)
    for _ in range(4):
        again = _run(hk, x, tok, 20)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_no_rows(hk, cuda):
    import torch
    x = torch.empty((0, 50), device=cuda)
    tok = torch.empty(0, dtype=torch.int64, device=cuda)
    hk.token_logprob_fwd(x, tok, torch.empty(0, device=cuda), None, None, None, None, IGN)
    hk.token_logprob_bwd(x, tok, torch.empty(0, device=cuda), None, torch.empty(0, device=cuda), None, torch.empty_like(x), IGN)
