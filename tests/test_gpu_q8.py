"""GPU parity of activations kept in 8 bits (hk_q8_*) and of the norm whose input is kept that way (hk_add_ln_q8_*)."""
import math

import pytest

pytestmark = pytest.mark.gpu

TYPES = ("fp32", "bf16", "fp16")
EPS = 1e-6
# what rounds to an infinity lies half a step past the largest number: an fp16 row of one column, whose x - mu is the rounding to 8
# bits alone and whose rs is 1 / sqrt(eps), has gradients of that size
LARGEST = {"fp32": 2.0 ** 127, "bf16": 2.0 ** 127, "fp16": 65504.0 * (1 - 2.0 ** -11)}
HALF = {"fp32": 2.0 ** -24, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}


def _dt(name):
    import torch
    return {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}[name]


def _pow2(n):
    import torch
    return ((n.long() + 1023) << 52).view(torch.float64)


def _pack(x):
    """The format's definition on fp64 values of fp32 numbers: (q, scale)."""
    import torch
    rows, cols = x.shape
    nb = (cols + 31) // 32
    pad = torch.zeros((rows, nb * 32), dtype=torch.float64, device=x.device)
    pad[:, :cols] = x
    b = pad.view(rows, nb, 32)
    big = b.abs().amax(2)
    bad = ~torch.isfinite(b).all(2)
    e = ((torch.where(bad, torch.zeros_like(big), big).float().view(torch.int32) >> 23) & 255).clamp(min=7).long()
    q = torch.where(bad[..., None], torch.zeros_like(b), (b * _pow2(133 - e)[..., None])).round().clamp(-127, 127)
    e = torch.where(bad, torch.full_like(e, 255), e)
    return q.to(torch.int8).view(rows, nb * 32), e.to(torch.uint8), bad


def _values(q, scale, cols):
    import torch
    rows, nb = scale.shape
    v = q.double().view(rows, nb, 32) * _pow2(scale.long() - 133)[..., None]
    v = torch.where((scale == 255)[..., None], torch.full_like(v, math.nan), v)
    return v.reshape(rows, nb * 32)[:, :cols]


WIDTHS = [1, 2, 3, 5, 7, 8, 9, 31, 32, 33, 63, 64, 65, 100, 127, 256, 257, 512, 513, 1000, 1021, 2047, 4096, 8191]


def _check_kept(q, scale, x, what=""):
    import torch
    want_q, want_e, bad = _pack(x)
    assert torch.equal(scale, want_e), (what, (scale != want_e).nonzero()[:4])
    good = (~bad)[..., None].expand(*bad.shape, 32).reshape(q.shape)
    assert torch.equal(q[good], want_q[good]), (what, ((q != want_q) & good).nonzero()[:4])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", WIDTHS)
def test_pack_and_unpack_are_exact(hk, cuda, dtype, cols):
    import torch
    for rows in (1, 5, 67):
        g = torch.Generator(device=cuda).manual_seed(cols)
        x = (torch.randn((rows, cols), generator=g, device=cuda) *
             torch.exp2(torch.randint(-8, 9, (rows, cols), generator=g, device=cuda).float())).to(_dt(dtype))
        x[0, 0] = 0.0
        q, scale = hk.q8_empty(rows, cols, cuda)
        q.fill_(99)
        hk.q8_pack(x, q, scale)
        torch.cuda.synchronize()
        _check_kept(q, scale, x.float().double(), (dtype, rows, cols))
        for out_type in TYPES:
            out = torch.full((rows, cols), 7.0, device=cuda).to(_dt(out_type))
            hk.q8_unpack(q, scale, out)
            torch.cuda.synchronize()
            assert torch.equal(out, _values(q, scale, cols).float().to(_dt(out_type)))


def test_special_values(hk, cuda):
    import torch
    x = torch.zeros((1, 32 * 12), device=cuda)
    b = x.view(12, 32)
    b[0, 3] = math.nan
    b[1, 4] = math.inf
    b[2, 5] = -math.inf
    b[3, :] = torch.finfo(torch.float32).max
    b[4, :] = -torch.finfo(torch.float32).max
    b[5, :] = torch.finfo(torch.float32).tiny
    b[6, :] = 2.0 ** -149
    b[7, 0], b[7, 1], b[7, 2], b[7, 3] = 1.0, 0.5 / 64, 1.5 / 64, 2.5 / 64       # halves: to the even one
    b[8, 0], b[8, 1], b[8, 2] = 127.5 / 64, -127.49 / 64, -127.5 / 64            # cut, not wrapped
    b[9, :] = -0.0
    b[10, 0], b[10, 1] = 2.0 ** -118, 2.0 ** -126
    b[11, 7] = -math.nan
    q, scale = hk.q8_empty(1, x.shape[1], cuda)
    hk.q8_pack(x, q, scale)
    torch.cuda.synchronize()
    _check_kept(q, scale, x.double())
    assert q.view(12, 32)[8, :3].tolist() == [127, -127, -127] and q.view(12, 32)[7, :4].tolist() == [64, 0, 2, 2]
    out = torch.empty_like(x)
    hk.q8_unpack(q, scale, out)
    torch.cuda.synchronize()
    want = _values(q, scale, x.shape[1]).float()
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out.nan_to_num(), want.nan_to_num())
    # every exponent that the format has, those included that packing never gives
    scale = torch.arange(256, device=cuda).to(torch.uint8)[None]
    q = torch.randint(-127, 128, (1, 256 * 32), device=cuda).to(torch.int8)
    out = torch.empty((1, 256 * 32), device=cuda)
    hk.q8_unpack(q, scale, out)
    torch.cuda.synchronize()
    want = _values(q, scale, 256 * 32).float()
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("dtype", TYPES)
def test_pack_of_pitched_rows(hk, cuda, dtype):
    import torch
    wide = torch.randn((19, 640), device=cuda).to(_dt(dtype))
    for first, cols in ((0, 96), (1, 96), (3, 101), (5, 7), (8, 600)):
        x = wide[:, first:first + cols]
        q, scale = hk.q8_empty(19, cols, cuda)
        hk.q8_pack(x, q, scale)
        torch.cuda.synchronize()
        _check_kept(q, scale, x.float().double())
        out = torch.full((19, cols + 9), 3.0, device=cuda).to(x.dtype)
        hk.q8_unpack(q, scale, out[:, 4:4 + cols])
        torch.cuda.synchronize()
        assert torch.equal(out[:, 4:4 + cols], _values(q, scale, cols).float().to(x.dtype))
        assert bool((out[:, :4] == 3).all()) and bool((out[:, 4 + cols:] == 3).all())


# ------------------------------- the norm -----------------------------------
def _norm_inputs(rows, cols, dtype, rtype, seed):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(std=1.0, mean=0.0, dt=dtype, shape=(rows, cols)):
        return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(_dt(dt))
    x0 = normal(1.0, 0.3)
    res = normal(2.0, 0.1, rtype) if rtype else None
    gamma = (torch.rand(cols, generator=g, device="cuda") * 0.8 + 0.6).to(_dt(dtype))
    beta = normal(0.2, shape=(cols,))
    return x0, res, gamma, beta, normal


def _forward(hk, x0, res, gamma, beta, rms, with_sum=True, fill=7.0):
    import torch
    rows, cols = x0.shape
    z = torch.full_like(x0, fill)
    s = torch.full_like(res, fill) if res is not None and with_sum else None
    q, scale = hk.q8_empty(rows, cols, x0.device)
    mu, rs = torch.full((rows,), fill, device=x0.device), torch.full((rows,), fill, device=x0.device)
    hk.add_ln_q8_fwd(x0, res, gamma, beta, z, s, q, scale, mu, rs, EPS, rms)
    torch.cuda.synchronize()
    return z, s, q, scale, mu, rs


def _moments64(x, rms):
    mu = x.mean(1)
    var = (x * x).mean(1) if rms else ((x - mu[:, None]) ** 2).mean(1)
    return mu, 1 / (var + EPS).sqrt()


def _store(v, dtype):
    """What rounding to the storage type may add: half a step, and half a step of the smallest numbers for fp16."""
    return v.abs() * HALF[dtype] + (2.0 ** -25 if dtype == "fp16" else 2.0 ** -140)


def _check_forward(out, x0, res, gamma, beta, rms, dtype, rtype, what=""):
    """fp32 sums of n terms, at most 64 to a thread and 12 levels of merges: 76 * 2^-24 < 2^-17.7 of the terms' magnitudes."""
    import torch
    z, s, q, scale, mu, rs = out
    x = x0.float() if res is None else x0.float() + res.float()
    if s is not None:
        assert torch.equal(s, x.to(s.dtype)), what
    x = x.double()
    _check_kept(q, scale, x, what)
    m, r = _moments64(x, rms)
    size = x.abs().mean(1)
    assert bool(((mu.double() - m).abs() <= 2.0 ** -17.7 * size + 2.0 ** -23 * m.abs()).all()), what
    # rs: the mean square is off by 2^-17.7 of itself (LayerNorm also by the mean's error, 2^-17.7 size of every deviation,
    # whose square's mean is second order), half of which reaches the root; root, division and eps 2^-22
    dev = (2.0 ** -17.7 * size) ** 2 * r * r
    tr = 2.0 ** -18.7 + 2.0 ** -22 + dev
    assert bool(((rs.double() - r).abs() <= tr * r).all()), (what, float(((rs.double() - r).abs() / r).max()))
    g = 1.0 if gamma is None else gamma.double()
    b = 0.0 if beta is None else beta.double()
    n = (x if rms else x - m[:, None]) * r[:, None]
    want = g * n + b
    e = abs(g) * (n.abs() * (tr + 2.0 ** -22)[:, None] + (0 if rms else (2.0 ** -17.7 * size * r)[:, None]))
    bound = e + 2.0 ** -23 * (want.abs() + abs(b)) + _store(want, dtype)
    assert bool(((z.double() - want).abs() <= bound).all()), (what, float(((z.double() - want).abs() / bound).max()))


NORM_WIDTHS = [1, 2, 5, 8, 9, 33, 64, 65, 127, 128, 256, 250, 511, 512, 600, 1000, 1021, 1536, 2048, 2500, 4096, 5120, 8191]
COMBOS = [("fp32", ""), ("fp32", "fp32"), ("bf16", ""), ("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp16", "fp32")]


@pytest.mark.parametrize("dtype,rtype", COMBOS)
@pytest.mark.parametrize("rms", [True, False])
def test_norm_forward(hk, cuda, dtype, rtype, rms):
    import torch
    for cols in NORM_WIDTHS:
        for rows in (1, 7, 70):
            x0, res, gamma, beta, _ = _norm_inputs(rows, cols, dtype, rtype, rows + cols)
            b = None if rms else beta
            out = _forward(hk, x0, res, gamma, b, rms)
            _check_forward(out, x0, res, gamma, b, rms, dtype, rtype, (dtype, rtype, rms, rows, cols))
            z, _, q, scale, mu, rs = out
            again = torch.full_like(z, 7.0)
            hk.add_ln_q8_out(q, scale, mu, rs, gamma, b, again, rms)
            x8 = _values(q, scale, cols)
            n = (x8 if rms else x8 - mu.double()[:, None]) * rs.double()[:, None]
            want = gamma.double() * n + (0.0 if rms else beta.double())
            shift = 0 if rms else (mu.double().abs() * rs.double())[:, None] * gamma.double().abs()
            bound = 2.0 ** -22 * (want.abs() + (gamma.double() * n).abs() + shift) + _store(want, dtype)
            assert bool(((again.double() - want).abs() <= bound).all()), (dtype, rtype, rms, rows, cols)


def _backward(hk, dz, up, q, scale, mu, rs, gamma, rms, with_dres, weights=True):
    import torch
    dx = torch.full_like(dz, 7.0)
    dres = torch.full_like(up if up is not None else dz, 7.0) if with_dres else None
    dg = torch.full((dz.shape[1],), 7.0, device=dz.device).to(dz.dtype) if weights else None
    db = torch.full_like(dg, 7.0) if weights and not rms else None
    hk.add_ln_q8_bwd(dz, up, q, scale, mu, rs, gamma, dx, dres, dg, db, rms)
    torch.cuda.synchronize()
    return dx, dres, dg, db


def _check_backward(got, dz, up, q, scale, mu, rs, gamma, rms, dtype, rtype, what=""):
    """x^ is off by 2^-22 (|x^| + |mu| rs) from its two operations; the row sums of n terms by 2^-17.7 of the terms' magnitudes (as in
    the forward) on top of x^'s; three operations of 2^-24 follow.  Column sums: a thread adds at most one row in 128 of the rows
    one after the other, the partial sums meet in some 16 steps or in 64 bits: (rows / 128 + 32) 2^-24 of the terms."""
    import torch
    dx, dres, dg, db = got
    rows, cols = dz.shape
    x8 = _values(q, scale, cols)
    m, r = mu.double()[:, None], rs.double()[:, None]
    n = (x8 if rms else x8 - m) * r
    en = 2.0 ** -22 * (n.abs() + (0 if rms else m.abs() * r))
    d = dz.double()
    u = d * (1.0 if gamma is None else gamma.double())
    k1 = 0.0 if rms else u.mean(1, keepdim=True)
    k2 = (u * n).mean(1, keepdim=True)
    want = r * (u - n * k2 - k1)
    ek2 = 2.0 ** -17.7 * (u * n).abs().mean(1, keepdim=True) + (u.abs() * en).mean(1, keepdim=True)
    ek1 = 0.0 if rms else 2.0 ** -17.7 * u.abs().mean(1, keepdim=True)
    bound = r * (n.abs() * ek2 + en * k2.abs() + ek1 + 2.0 ** -22 * (u.abs() + (n * k2).abs() + abs(k1)))
    if up is not None:
        want = want + up.double()
        bound = bound + 2.0 ** -23 * (want.abs() + up.double().abs())
    fits = want.abs() < LARGEST[dtype]
    assert bool(((dx.double() - want).abs() <= bound + _store(want, dtype))[fits].all()), \
        (what, float(((dx.double() - want).abs() / (bound + _store(want, dtype)))[fits].max()))
    assert bool((dx.double() == want.sign() * math.inf)[want.abs() > LARGEST[dtype] * 1.01].all()), what
    if dres is not None:
        fits = want.abs() < LARGEST[rtype or dtype]
        assert bool(((dres.double() - want).abs() <= bound + _store(want, rtype or dtype))[fits].all()), what
    chain = (rows / 128 + 32) * 2.0 ** -24
    if dg is not None:
        want = (d * n).sum(0)
        bound = chain * (d * n).abs().sum(0) + (d.abs() * en).sum(0) + _store(want, dtype)
        assert bool(((dg.double() - want).abs() <= bound).all()), (what, float(((dg.double() - want).abs() / bound).max()))
    if db is not None:
        want = d.sum(0)
        assert bool(((db.double() - want).abs() <= chain * d.abs().sum(0) + _store(want, dtype)).all()), what


@pytest.mark.parametrize("dtype,rtype", COMBOS)
@pytest.mark.parametrize("rms", [True, False])
def test_norm_backward(hk, cuda, dtype, rtype, rms):
    for cols in NORM_WIDTHS:
        for rows in (1, 7, 70):
            x0, res, gamma, beta, normal = _norm_inputs(rows, cols, dtype, rtype, rows * cols)
            _, _, q, scale, mu, rs = _forward(hk, x0, res, gamma, None if rms else beta, rms)
            dz = normal()
            up = normal(dt=rtype) if rtype else None
            got = _backward(hk, dz, up, q, scale, mu, rs, gamma, rms, bool(rtype))
            _check_backward(got, dz, up, q, scale, mu, rs, gamma, rms, dtype, rtype, (dtype, rtype, rms, rows, cols))


@pytest.mark.parametrize("dtype,cols", [("bf16", 16384), ("bf16", 20011), ("bf16", 32768), ("fp32", 16385), ("fp32", 32768),
                                        ("fp16", 32767)])
def test_wide_rows(hk, cuda, dtype, cols):
    for rms in (True, False):
        x0, res, gamma, beta, normal = _norm_inputs(9, cols, dtype, "fp32", cols)
        b = None if rms else beta
        out = _forward(hk, x0, res, gamma, b, rms)
        _check_forward(out, x0, res, gamma, b, rms, dtype, "fp32", (dtype, cols))
        dz, up = normal(), normal(dt="fp32")
        got = _backward(hk, dz, up, *out[2:], gamma, rms, True)
        _check_backward(got, dz, up, *out[2:], gamma, rms, dtype, "fp32", (dtype, cols))


@pytest.mark.parametrize("dtype,rtype,cols", [("bf16", "bf16", 12288), ("bf16", "bf16", 17001), ("fp16", "fp32", 9000),
                                              ("fp32", "fp32", 16384), ("fp16", "", 20000), ("fp32", "fp32", 20011)])
def test_wide_rows_of_a_batch(hk, cuda, dtype, rtype, cols):
    """Wide rows, more of them than the one-launch backward takes: against the formula, and over what the gradients are made of."""
    import torch
    for rms in (True, False):
        x0, res, gamma, beta, normal = _norm_inputs(1100, cols, dtype, rtype, cols)
        out = _forward(hk, x0, res, gamma, None, rms)
        dz, up = normal(), normal(dt=rtype) if rtype else None
        got = _backward(hk, dz, up, *out[2:], gamma, rms, bool(rtype))
        _check_backward(got, dz, up, *out[2:], gamma, rms, dtype, rtype or dtype, (dtype, cols, rms))
        a, b = dz.clone(), up.clone() if rtype else None
        dg, db = torch.empty_like(gamma), None if rms else torch.empty_like(gamma)
        hk.add_ln_q8_bwd(a, b, *out[2:], gamma, a, b, dg, db, rms)
        assert torch.equal(a, got[0]) and (b is None or torch.equal(b, got[1])) and torch.equal(dg, got[2])
        assert rms or torch.equal(db, got[3])
        dx = torch.empty_like(dz)
        hk.add_ln_q8_bwd(dz, up, *out[2:], gamma, dx, None, None, None, rms)      # without the sums
        assert torch.equal(dx, got[0])


@pytest.mark.parametrize("rows,cols", [(5000, 96), (3001, 1021), (2600, 4096), (9000, 64), (40000, 8)])
def test_many_rows(hk, cuda, rows, cols):
    """More rows than workgroups: the backward's workgroups walk."""
    for dtype, rtype, rms in (("bf16", "bf16", True), ("bf16", "", False), ("fp32", "fp32", True)):
        x0, res, gamma, beta, normal = _norm_inputs(rows, cols, dtype, rtype, rows)
        b = None if rms else beta
        out = _forward(hk, x0, res, gamma, b, rms)
        _check_forward(out, x0, res, gamma, b, rms, dtype, rtype, (dtype, rows, cols))
        dz, up = normal(), normal(dt=rtype) if rtype else None
        got = _backward(hk, dz, up, *out[2:], gamma, rms, False)
        _check_backward(got, dz, up, *out[2:], gamma, rms, dtype, rtype, (dtype, rows, cols))


def test_optional_operands(hk, cuda):
    import torch
    x0, res, gamma, beta, normal = _norm_inputs(12, 300, "bf16", "fp32", 5)
    for g in (gamma, None):
        for b in (beta, None):
            out = _forward(hk, x0, res, g, b, False, with_sum=False)
            _check_forward(out, x0, res, g, b, False, "bf16", "fp32")
    out = _forward(hk, x0, None, gamma, None, True)
    dz, up = normal(), normal(dt="fp32")
    full = _backward(hk, dz, up, *out[2:], gamma, True, True)
    dx = torch.empty_like(dz)
    hk.add_ln_q8_bwd(dz, up, *out[2:], gamma, dx, None, None, None, True)                 # no weights, no workspace
    assert torch.equal(dx, full[0])
    dres = torch.empty_like(up)
    hk.add_ln_q8_bwd(dz, None, *out[2:], None, dx, dres, None, None, True)                # no upstream gradient, no gamma
    _check_backward((dx, dres, None, None), dz, None, *out[2:], None, True, "bf16", "fp32")
    ln = _forward(hk, x0, None, gamma, beta, False)
    dg, db = torch.empty_like(gamma), torch.empty_like(gamma)
    hk.add_ln_q8_bwd(dz, None, *ln[2:], gamma, dx, None, dg, None, False)
    hk.add_ln_q8_bwd(dz, None, *ln[2:], gamma, dx, None, None, db, False)
    _check_backward((dx, None, dg, db), dz, None, *ln[2:], gamma, False, "bf16", "")
    hk.add_ln_q8_bwd(dz, up, out[2], out[3], None, out[5], gamma, dx, None, None, None, True)   # an RMSNorm needs no mu
    assert torch.equal(dx, full[0])


def test_in_place(hk, cuda):
    """The sum over the residual or x0, the gradients over dz and the upstream gradient."""
    import torch
    for dtype, rtype, cols in (("bf16", "bf16", 4096), ("bf16", "fp32", 1000), ("fp32", "fp32", 513), ("bf16", "bf16", 5003)):
        x0, res, gamma, beta, normal = _norm_inputs(300, cols, dtype, rtype, cols)
        out = _forward(hk, x0, res, gamma, None, True)
        stream = res.clone()
        z = torch.empty_like(x0)
        q, scale = hk.q8_empty(300, cols, cuda)
        mu, rs = torch.empty(300, device=cuda), torch.empty(300, device=cuda)
        hk.add_ln_q8_fwd(x0, stream, gamma, None, z, stream, q, scale, mu, rs, EPS, True)
        assert all(torch.equal(a, b) for a, b in zip((z, stream, q, scale, mu, rs), out))
        if dtype == rtype:
            other = x0.clone()
            hk.add_ln_q8_fwd(other, res, gamma, None, z, other, q, scale, mu, rs, EPS, True)
            assert all(torch.equal(a, b) for a, b in zip((z, other, q, scale, mu, rs), out))
        dz, up = normal(), normal(dt=rtype)
        full = _backward(hk, dz, up, *out[2:], gamma, True, True)
        dg = torch.empty_like(gamma)
        a, b = dz.clone(), up.clone()
        hk.add_ln_q8_bwd(a, b, *out[2:], gamma, a, b, dg, None, True)
        assert torch.equal(a, full[0]) and torch.equal(b, full[1])
        _check_backward((a, b, dg, None), dz, up, *out[2:], gamma, True, dtype, rtype)     # (its sums in another order)


@pytest.mark.parametrize("cols", [256, 1000, 1021])
def test_pitched_rows(hk, cuda, cols):
    import torch
    rows = 41

    def wide(dt):
        return torch.randn((rows, cols + 50), device=cuda).to(_dt(dt))
    for dtype, rtype in (("bf16", "fp32"), ("fp16", "fp16"), ("fp32", "fp32")):
        for first in (0, 1, 16):
            x0, res, z, s = (wide(t)[:, first:first + cols] for t in (dtype, rtype, dtype, rtype))
            gamma = torch.rand(cols, device=cuda).to(_dt(dtype)) + 0.5
            q, scale = hk.q8_empty(rows, cols, cuda)
            mu, rs = torch.empty(rows, device=cuda), torch.empty(rows, device=cuda)
            hk.add_ln_q8_fwd(x0, res, gamma, None, z, s, q, scale, mu, rs, EPS, True)
            dense = _forward(hk, x0.contiguous(), res.contiguous(), gamma, None, True)
            assert all(torch.equal(a, b) for a, b in zip((z, s, q, scale, mu, rs), dense))
            dz, up, dx, dres = (wide(t)[:, first:first + cols] for t in (dtype, rtype, dtype, rtype))
            dg = torch.empty_like(gamma)
            hk.add_ln_q8_bwd(dz, up, q, scale, mu, rs, gamma, dx, dres, dg, None, True)
            ref = _backward(hk, dz.contiguous(), up.contiguous(), q, scale, mu, rs, gamma, True, True)
            assert torch.equal(dx, ref[0]) and torch.equal(dres, ref[1]) and torch.equal(dg, ref[2])
            base = torch.full((rows, cols + 50), 3.0, device=cuda).to(_dt(dtype))
            hk.add_ln_q8_out(q, scale, mu, rs, gamma, None, base[:, first + 1:first + 1 + cols], True)
            assert bool((base[:, :first + 1] == 3).all()) and bool((base[:, first + 1 + cols:] == 3).all())


@pytest.mark.parametrize("dtype,rtype", [("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "fp32"), ("fp16", "")])
@pytest.mark.parametrize("cols", [2057, 2560, 3579, 4095, 4096, 8200, 9001, 17001])
def test_rows_on_odd_elements(hk, cuda, dtype, rtype, cols):
    """Rows of 16-bit elements that begin on odd ones, between columns of NaN, give what the same rows on 16-byte boundaries
    give, bit by bit; also where the gradients are written over what they are made of."""
    import torch
    gen = torch.Generator(device=cuda).manual_seed(cols)
    for rows, places in ((37, ((1, 4, 1, 2), (0, 1, 3, 0))), (1300, ((1, 1, 3, 8),))):
        whole = (cols + 7) // 8 * 8 + 16
        data = [torch.randn((rows, cols), generator=gen, device=cuda).to(_dt(t)) if t else None for t in (dtype, rtype, dtype, rtype)]
        gamma = (torch.rand(cols, generator=gen, device=cuda) + 0.5).to(_dt(dtype))
        sides = []
        for place in ((8, 8, 8, 8),) + places:
            def rows_at(first, value, t):
                if value is None and t is None:
                    return None
                width = whole if place[0] == 8 else whole + 1 + place[3] % 2
                out = torch.full((rows, width), math.nan, device=cuda, dtype=_dt(t) if t else value.dtype)[:, first:first + cols]
                if value is not None:
                    out.copy_(value)
                return out
            x0, res, dz, up = (rows_at(f, v, None) for f, v in zip(place, data))
            z, dx = rows_at(place[2], None, dtype), rows_at(place[1], None, dtype)
            s = rows_at(place[0], None, rtype) if rtype else None
            q, scale = hk.q8_empty(rows, cols, cuda)
            mu, rs, dg = torch.empty(rows, device=cuda), torch.empty(rows, device=cuda), torch.empty_like(gamma)
            hk.add_ln_q8_fwd(x0, res, gamma, None, z, s, q, scale, mu, rs, EPS, True)
            hk.add_ln_q8_bwd(dz, up, q, scale, mu, rs, gamma, dx, None, dg, None, True)
            kept = [t.clone() for t in (z, q, scale, mu, rs, dx, dg)] + ([s.clone()] if rtype else [])
            if rtype and rows > 1024:
                hk.add_ln_q8_bwd(dz, up, q, scale, mu, rs, gamma, dz, up, dg, None, True)
                assert torch.equal(dz, dx) and torch.equal(up, dx if rtype == dtype else up) and torch.equal(dg, kept[6])
            if rtype:
                hk.add_ln_q8_fwd(x0, res, gamma, None, z, res, q, scale, mu, rs, EPS, True)
                assert torch.equal(res, s) and torch.equal(z, kept[0])
            sides.append(kept)
        for other in sides[1:]:
            assert all(torch.equal(a, b) for a, b in zip(sides[0], other))


def test_rows_with_nan_stay_by_themselves(hk, cuda):
    """A row that holds a NaN gives NaN in its own row; the other rows' results are as without it."""
    import torch
    for cols in (64, 1000, 4096, 1021):
        x0, _, gamma, _, normal = _norm_inputs(40, cols, "bf16", "", cols)
        clean = _forward(hk, x0, None, gamma, None, True)
        dz = normal()
        ref = _backward(hk, dz, None, *clean[2:], gamma, True, False, weights=False)
        x0[7, 3] = math.nan
        out = _forward(hk, x0, None, gamma, None, True)
        rest = torch.arange(40, device=cuda) != 7
        assert all(torch.equal(a[rest], b[rest]) for a, b in zip(out, clean) if a is not None)
        assert bool(torch.isnan(out[0][7]).all()) and int(out[3][7, 0]) == 255
        got = _backward(hk, dz, None, *out[2:], gamma, True, False, weights=False)
        assert torch.equal(got[0][rest], ref[0][rest]) and bool(torch.isnan(got[0][7]).all())


def test_gradient_against_differences(hk, cuda):
    """Differences of the restored norm: x8 moved by steps of its format, fp32 arithmetic in 64 bits around it."""
    import torch
    rows, cols = 2, 37
    for rms in (True, False):
        x0, _, gamma, beta, normal = _norm_inputs(rows, cols, "fp32", "", 3)
        _, _, q, scale, mu, rs = _forward(hk, x0, None, gamma, None if rms else beta, rms)
        x8 = _values(q, scale, cols)
        # statistics of the kept values themselves, so that the function that is differentiated is the norm of x8
        m, r = _moments64(x8, rms)
        mu, rs = m.float(), r.float()
        w = normal()

        def loss(v):
            mm, rr = _moments64(v, rms)
            return ((v if rms else v - mm[:, None]) * rr[:, None] * gamma.double() * w.double()).sum(1)
        dx, _, dg, _ = _backward(hk, w, None, q, scale, mu, rs, gamma, rms, False)
        h = 1e-4
        for c in range(cols):
            up, down = x8.clone(), x8.clone()
            up[:, c] += h
            down[:, c] -= h
            diff = (loss(up) - loss(down)) / (2 * h)
            # the difference's own error: h^2 / 6 of a third derivative below 1e3, and 2^-52 of sums below 100 over h;
            # the kernel's: 2^-17 of terms below 10, and eps against rs^2, whose share is below 1e-5
            assert bool(((diff - dx[:, c].double()).abs() <= 1e-5 + 2.0 ** -17 * 10 + 1e-4).all()), (rms, c)


def test_replayed_graph(hk, cuda):
    import torch
    x0, res, gamma, beta, normal = _norm_inputs(700, 1000, "bf16", "fp32", 1)
    rows, cols = x0.shape
    dz, up = normal(), normal(dt="fp32")
    z, s, zz, dx, dres = (torch.empty_like(t) for t in (x0, res, x0, x0, res))
    q, scale = hk.q8_empty(rows, cols, cuda)
    mu, rs = torch.empty(rows, device=cuda), torch.empty(rows, device=cuda)
    dg, db = torch.empty_like(gamma), torch.empty_like(gamma)
    ws = torch.empty(hk.add_ln_q8_bwd_workspace_bytes(rows, cols) // 4 + 4, device=cuda)

    def call():
        hk.add_ln_q8_fwd(x0, res, gamma, beta, z, s, q, scale, mu, rs, EPS, False)
        hk.add_ln_q8_out(q, scale, mu, rs, gamma, beta, zz, False)
        hk.add_ln_q8_bwd(dz, up, q, scale, mu, rs, gamma, dx, dres, dg, db, False, workspace=ws)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call()
    outs = (z, s, q, scale, mu, rs, zz, dx, dres, dg, db)
    for turn in range(3):
        x0.copy_(torch.randn(x0.shape, device=cuda) * (turn + 1))
        dz.copy_(torch.randn(x0.shape, device=cuda))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, outs))


def test_no_rows(hk, cuda):
    import torch
    x = torch.empty((0, 64), device=cuda)
    q, scale = hk.q8_empty(0, 64, cuda)
    none = torch.empty(0, device=cuda)
    hk.q8_pack(x, q, scale)
    hk.q8_unpack(q, scale, x)
    hk.add_ln_q8_fwd(x, None, None, None, x, None, q, scale, none, none, EPS, True)
    dg = torch.ones(64, device=cuda)
    db = torch.ones(64, device=cuda)
    hk.add_ln_q8_bwd(x, None, q, scale, none, none, None, x, None, dg, db, False)
    torch.cuda.synchronize()
    assert bool((dg == 0).all()) and bool((db == 0).all())        # the empty sums
