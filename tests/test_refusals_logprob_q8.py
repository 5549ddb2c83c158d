"""What the token log probability and 8-bit checkpoint entry points refuse, before anything reaches a GPU."""
import ctypes
import importlib

import pytest

import helpers  # noqa: F401  (paths)


@pytest.fixture()
def lib(hk):
    return hk.lib()


BUF = ctypes.create_string_buffer(1 << 12)
ADDR = (ctypes.addressof(BUF) + 63) // 64 * 64
P = ctypes.c_void_p(ADDR)
ODD = ctypes.c_void_p(ADDR + 4)
NULL = ctypes.c_void_p(0)


def i64(v):
    return ctypes.c_int64(v)


def size(v):
    return ctypes.c_size_t(v)


def _forward(lib, dtype=6, logits=P, pitch=64, tokens=P, logprob=P, entropy=P, lse=P, value=NULL, token=NULL, top=0, rows=4,
             cols=64, ws=NULL, wsb=0):
    return lib.hk_token_logprob_fwd(dtype, logits, i64(pitch), tokens, logprob, entropy, lse, value, token, i64(top), i64(rows),
                                    i64(cols), i64(-100), ws, size(wsb), NULL)


@pytest.mark.parametrize("change,code,word", [
    (dict(dtype=7), -2, b"dtype"), (dict(dtype=4), -2, b"dtype"), (dict(rows=-1), -1, b"shape"), (dict(cols=0), -1, b"shape"),
    (dict(cols=1 << 31, pitch=1 << 31), -1, b"31 bits"), (dict(rows=1 << 31), -1, b"31 bits"),
    (dict(logits=NULL), -1, b"null"), (dict(tokens=NULL), -1, b"null"),
    (dict(logprob=NULL, entropy=NULL, lse=NULL), -1, b"null"), (dict(pitch=63), -1, b"pitch"),
    (dict(top=33, value=P, token=P), -1, b"at most 32"), (dict(top=-1), -1, b"shape"), (dict(top=2), -1, b"null alternatives"),
    (dict(top=2, value=P), -1, b"null alternatives"), (dict(rows=1, cols=60000, pitch=60000), -4, b"workspace"),
    (dict(rows=1, cols=60000, pitch=60000, ws=ODD, wsb=1 << 11), -1, b"boundary")])
def test_forward(lib, change, code, word):
    assert _forward(lib, **change) == code
    assert word in lib.hk_last_error(), lib.hk_last_error()


def test_forward_of_no_rows_needs_nothing(lib):
    assert _forward(lib, rows=0, logits=NULL, tokens=NULL, logprob=NULL) == 0


def test_workspace_questions(hk, lib):
    n = ctypes.c_size_t(5)
    assert lib.hk_token_logprob_workspace_bytes(6, i64(4), i64(0), i64(0), ctypes.byref(n)) == -1
    assert lib.hk_token_logprob_workspace_bytes(7, i64(4), i64(8), i64(0), ctypes.byref(n)) == -2
    assert lib.hk_token_logprob_workspace_bytes(6, i64(4), i64(8), i64(33), ctypes.byref(n)) == -1
    assert lib.hk_token_logprob_workspace_bytes(6, i64(4), i64(8), i64(3), None) == -1
    assert lib.hk_add_ln_q8_bwd_workspace_bytes(i64(4), i64(40000), ctypes.byref(n)) == -1
    assert lib.hk_add_ln_q8_bwd_workspace_bytes(i64(4), i64(8), None) == -1
    for dt in (5, 6, 8):
        for rows in (0, 1, 3, 255, 256, 1000, 1 << 20):
            for cols in (1, 7, 4096, 50257, 131072, 1 << 20, (1 << 31) - 16):
                for top in (0, 1, 32):
                    # parts of few long rows: at most 8 of them, 12 bytes an alternative and 16 of statistics
                    assert 0 <= hk.token_logprob_workspace_bytes(dt, rows, cols, top) <= 8 * rows * (12 * top + 16)


def _backward(lib, dtype=6, logits=P, pitch=64, tokens=P, lse=P, entropy=P, g=P, h=P, out=P, out_pitch=64, rows=4, cols=64,
              start=0):
    return lib.hk_token_logprob_bwd(dtype, logits, i64(pitch), tokens, lse, entropy, g, h, out, i64(out_pitch), i64(rows),
                                    i64(cols), i64(start), i64(-100), NULL)


@pytest.mark.parametrize("change,code,word", [
    (dict(dtype=7), -2, b"dtype"), (dict(rows=-1), -1, b"shape"), (dict(start=-1), -1, b"shape"), (dict(lse=NULL), -1, b"null"),
    (dict(out=NULL), -1, b"null"), (dict(g=NULL, h=NULL), -1, b"null"), (dict(entropy=NULL), -1, b"entropy"),
    (dict(pitch=10), -1, b"pitch"), (dict(out_pitch=10), -1, b"pitch")])
def test_backward(lib, change, code, word):
    assert _backward(lib, **change) == code
    assert word in lib.hk_last_error(), lib.hk_last_error()


@pytest.mark.parametrize("change,word", [
    (dict(shards=0), b"shape"), (dict(shards=65), b"64 shards"), (dict(top=33), b"32 alternatives"), (dict(top=1), b"null alternatives"),
    (dict(stats=NULL), b"null"), (dict(tokens=NULL), b"null"), (dict(lp=NULL), b"null"), (dict(rows=-2), b"shape")])
def test_combine(lib, change, word):
    a = dict(stats=P, tokens=P, lp=P, shards=2, top=0, rows=4)
    a.update(change)
    rc = lib.hk_vocab_parallel_logprob_combine(a["stats"], NULL, NULL, i64(a["shards"]), a["tokens"], i64(-100), i64(-1), a["lp"],
                                               NULL, NULL, NULL, NULL, i64(a["top"]), i64(a["rows"]), NULL)
    assert rc == -1 and word in lib.hk_last_error(), lib.hk_last_error()


def test_stats(lib):
    rc = lib.hk_vocab_parallel_logprob_stats(6, P, i64(64), P, NULL, NULL, NULL, i64(0), i64(4), i64(64), i64(0), i64(-100), NULL,
                                             size(0), NULL)
    assert rc == -1 and b"null output" in lib.hk_last_error()
    rc = lib.hk_vocab_parallel_logprob_stats(6, P, i64(64), P, P, NULL, NULL, i64(0), i64(4), i64(64), i64(-5), i64(-100), NULL,
                                             size(0), NULL)
    assert rc == -1 and b"vocab_start" in lib.hk_last_error()


def test_kept_values(lib):
    for f in (lib.hk_q8_pack,):
        assert f(7, P, i64(64), P, P, i64(4), i64(64), NULL) == -2
        assert f(6, P, i64(10), P, P, i64(4), i64(64), NULL) == -1 and b"pitch" in lib.hk_last_error()
        assert f(6, P, i64(64), ODD, P, i64(4), i64(64), NULL) == -1 and b"8-byte" in lib.hk_last_error()
        assert f(6, NULL, i64(64), P, P, i64(4), i64(64), NULL) == -1 and b"null" in lib.hk_last_error()
        assert f(6, P, i64(64), P, P, i64(-4), i64(64), NULL) == -1
        assert f(6, NULL, i64(64), NULL, NULL, i64(0), i64(64), NULL) == 0
    assert lib.hk_q8_unpack(7, P, P, P, i64(64), i64(4), i64(64), NULL) == -2
    assert lib.hk_q8_unpack(6, ODD, P, P, i64(64), i64(4), i64(64), NULL) == -1
    assert lib.hk_q8_unpack(6, P, P, P, i64(6), i64(4), i64(64), NULL) == -1
    assert lib.hk_q8_unpack(6, P, P, NULL, i64(64), i64(4), i64(64), NULL) == -1


def _norm(lib, which, itype=8, rtype=6, rows=4, cols=64, pitch=64, q=P, x0=P, z=P, mu=P, rms=1, dbeta=NULL, wsb=1 << 20, ws=P):
    if which == "fwd":
        return lib.hk_add_ln_q8_fwd(itype, rtype, x0, i64(pitch), P, i64(64), P, NULL, z, i64(64), P, i64(64), q, P, mu, P, i64(rows),
                                    i64(cols), ctypes.c_float(1e-6), rms, NULL)
    if which == "out":
        return lib.hk_add_ln_q8_out(itype, q, P, mu, P, P, NULL, z, i64(pitch), i64(rows), i64(cols), rms, NULL)
    return lib.hk_add_ln_q8_bwd(itype, rtype, x0, i64(pitch), P, i64(64), q, P, mu, P, P, z, i64(64), P, i64(64), P, dbeta, i64(rows),
                                i64(cols), rms, ws, size(wsb), NULL)


@pytest.mark.parametrize("which", ["fwd", "out", "bwd"])
def test_norms(lib, which):
    assert _norm(lib, which, itype=7) == -2
    assert _norm(lib, which, cols=32769, pitch=32769) == -1 and b"32768" in lib.hk_last_error()
    assert _norm(lib, which, pitch=8) == -1 and b"pitch" in lib.hk_last_error()
    assert _norm(lib, which, q=ODD) == -1 and b"8-byte" in lib.hk_last_error()
    assert _norm(lib, which, z=NULL) == -1 and b"null" in lib.hk_last_error()
    assert _norm(lib, which, mu=NULL, rms=0) == -1 and b"null" in lib.hk_last_error()
    assert _norm(lib, which, rows=-1) == -1
    assert _norm(lib, which, rows=0, z=NULL, cols=0) == 0
    if which != "out":
        assert _norm(lib, which, itype=8, rtype=5) == -2 and b"residual" in lib.hk_last_error()
        assert _norm(lib, which, itype=6, rtype=8) == -2
        assert _norm(lib, which, x0=NULL) == -1
    if which == "bwd":
        assert _norm(lib, which, dbeta=P, rms=1) == -1 and b"no beta" in lib.hk_last_error()
        assert _norm(lib, which, wsb=16) == -4 and b"workspace" in lib.hk_last_error()
        assert _norm(lib, which, ws=ODD) == -1 and b"16-byte" in lib.hk_last_error()


def test_tensors_on_the_host_are_refused(hk):
    """The harness hands device pointers on: a tensor elsewhere is refused by name."""
    import torch
    x = torch.zeros(4, 64)
    tok = torch.zeros(4, dtype=torch.int64)
    v = torch.zeros(4)
    q, scale = hk.q8_empty(4, 64, "cpu")
    for call in (lambda: hk.token_logprob_fwd(x, tok, v, None, None, None, None, -100),
                 lambda: hk.token_logprob_bwd(x, tok, v, None, v, None, x, -100),
                 lambda: hk.vocab_parallel_logprob_stats(x, tok, torch.zeros(4, 4), None, None, 0, -100),
                 lambda: hk.vocab_parallel_logprob_combine(torch.zeros(2, 4, 4), None, None, tok, -100, v, None, None, None, None),
                 lambda: hk.q8_pack(x, q, scale), lambda: hk.q8_unpack(q, scale, x),
                 lambda: hk.add_ln_q8_fwd(x, None, None, None, x, None, q, scale, v, v, 1e-6, True),
                 lambda: hk.add_ln_q8_out(q, scale, v, v, None, None, x, True),
                 lambda: hk.add_ln_q8_bwd(x, None, q, scale, v, v, None, x, None, None, None, True)):
        with pytest.raises(hk.HkError, match="GPU"):
            call()
    with pytest.raises(hk.HkError, match="come together"):
        hk.token_logprob_fwd(x, tok, v, None, None, torch.zeros(4, 2), None, -100)
    with pytest.raises(hk.HkError, match="are asked for"):
        hk.vocab_parallel_logprob_combine(torch.zeros(2, 4, 4), None, None, tok, -100, v, None, None, torch.zeros(4, 2),
                                          torch.zeros(4, 2, dtype=torch.int64))


def test_operator_layer_refuses_host_arrays(hk):
    """The kernels are accelerator only; a missing array is an error, never a fault."""
    import torch
    ops = importlib.import_module("hotspa-ae_amd.hetu_ops")
    x, tok, v = torch.zeros(4, 64), torch.zeros(4, dtype=torch.int64), torch.zeros(4)
    q, scale = hk.q8_empty(4, 64, "cpu")
    for call in (lambda: ops.token_logprob(x, tok, v, None, None, None, None, -100), lambda: ops.q8_pack(x, q, scale),
                 lambda: ops.token_logprob_gradient(x, tok, v, None, v, None, x, -100), lambda: ops.q8_unpack(q, scale, x),
                 lambda: ops.vocab_parallel_logprob_stats(x, tok, torch.zeros(4, 4), None, None, 0, -100),
                 lambda: ops.add_ln_q8_fwd(x, None, None, None, x, None, q, scale, v, v, 1e-6, True),
                 lambda: ops.add_ln_q8_out(q, scale, v, v, None, None, x, True),
                 lambda: ops.add_ln_q8_bwd(x, None, q, scale, v, v, None, x, None, None, None, True)):
        with pytest.raises(ops.AssertionError_):
            call()
    for call in (lambda: ops.token_logprob(None, tok, v, None, None, None, None, -100), lambda: ops.q8_pack(None, q, scale),
                 lambda: ops.add_ln_q8_fwd(None, None, None, None, x, None, q, scale, v, v, 1e-6, True)):
        with pytest.raises(ops.HetuError):
            call()
    with pytest.raises(ops.HetuError):
        ops.add_ln_q8_fwd(x, None, None, None, None, None, None, None, None, None, 1e-6, True)
