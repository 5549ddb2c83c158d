"""The tail of a training step and the scoring of tokens, as cases that can be timed: log probabilities of given tokens
with entropy and top alternatives, their gradient, their vocabulary-parallel form, and norms whose input is kept in
8 bits for the backward pass.

A case is a dict of plain values; its "op" names the path, the other values its sizes and types.  `listed()` gives the
cases that are always measured, `draw(rng)` one more of the same ranges.  `prepare(case, seed)` makes what a program
holds before the call, `run(state)` is one pass: in elementary torch operations where `own` is false, through the
package's entry points where it is true.  `work(case)` is what a pass cannot do without, `exact(case, seed)` the
outputs from the definition in 64 bits.

Activations are kept as blocks of 32 columns with one power of two each (the MXINT8 format of the OCP microscaling
specification): values q * 2^(E - 133), q in [-127, 127], E the exponent field of the block's largest magnitude.
"""
import importlib
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
IGNORED = -100
BLOCK = 32
EPS = 1e-6
_PIECE = 1 << 27   # elements that one elementary operation of the plain form is given


def listed():
    return [
        # one step of a served model: log probability of the sampled token, 20 alternatives, one request
        {"name": "score_one", "op": "score", "rows": 1, "cols": 50257, "dtype": "bf16", "top": 20, "ignored": 0},
        # scoring of the tokens of a long batch with 8 alternatives each
        {"name": "score_batch", "op": "score", "rows": 16384, "cols": 32000, "dtype": "bf16", "top": 8, "ignored": 0},
        # gradient of a small model's policy loss over an odd vocabulary
        {"name": "grad_odd", "op": "grad", "rows": 96, "cols": 10007, "dtype": "fp32", "entropy": True, "ignored": 10},
        # gradient of a policy loss with an entropy bonus: the cross-entropy benchmark's shape
        {"name": "grad_batch", "op": "grad", "rows": 16384, "cols": 32000, "dtype": "bf16", "entropy": True,
         "ignored": 819},
        # one of 8 ranks' share of a decoding batch's scores, with alternatives
        {"name": "shard_small", "op": "shard", "rows": 64, "cols": 4000, "ranks": 8, "dtype": "fp16", "top": 5,
         "ignored": 0},
        # one of 4 ranks' share of a training batch: shards of an odd vocabulary, prompt tokens ignored
        {"name": "shard_batch", "op": "shard", "rows": 16384, "cols": 12565, "ranks": 4, "dtype": "bf16", "top": 0,
         "ignored": 1638},
        # an activation of a few tokens kept in 8 bits and restored
        {"name": "keep_small", "op": "keep", "rows": 128, "cols": 4096, "dtype": "bf16"},
        # the same of a training batch, at a width that is no multiple of a block
        {"name": "keep_batch", "op": "keep", "rows": 14549, "cols": 3579, "dtype": "fp32"},
        # LayerNorm on feature rows of an odd width whose input is kept in 8 bits
        {"name": "norm_odd", "op": "norm", "rows": 8191, "cols": 1021, "dtype": "fp16", "residual": "", "rms": False},
        # pre-norm block on 32768 packed tokens with an fp32 residual stream, its sum kept in 8 bits
        {"name": "norm_batch", "op": "norm", "rows": 32768, "cols": 4096, "dtype": "bf16", "residual": "fp32",
         "rms": True},
        # backward of a few tokens: the norm's output restored, gradients from the 8 bits
        {"name": "norm_grad_small", "op": "norm_grad", "rows": 512, "cols": 5120, "dtype": "bf16", "residual": "",
         "rms": False},
        # the same of 32768 packed tokens, with the upstream gradient of the residual stream
        {"name": "norm_grad_batch", "op": "norm_grad", "rows": 32768, "cols": 4096, "dtype": "bf16", "residual": "bf16",
         "rms": True},
    ]


# ---------------------------------------------------------------------------
# one more case of the same ranges
# ---------------------------------------------------------------------------
def _between(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high, odd):
    """A row width: with probability `odd` any number at all, else a multiple of 64."""
    n = _between(rng, low, high)
    return n if rng.random() < odd else max(64, n // 64 * 64)


def draw(rng):
    op = rng.choice(["score", "grad", "shard", "keep", "norm", "norm_grad"])
    dt = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    if op in ("score", "grad", "shard"):
        cols = _width(rng, 1000, 131072, 0.4)
        ranks = 1
        if op == "shard":
            ranks = rng.choice([2, 4, 8])
            cols = max(64, cols // ranks)
        rows = _between(rng, 1, max(1, min(16384, 8192 * 32000 // (cols * ranks))))
        case = {"op": op, "rows": rows, "cols": cols, "dtype": dt}
        if op == "shard":
            case["ranks"] = ranks
        if op == "grad":
            case["entropy"] = rng.random() < 0.6
        else:
            case["top"] = rng.choice([0, 1, 5, 20])
        case["ignored"] = 0 if case.get("top") else rows // 10
        return case
    cols = _width(rng, 64, 8192, 0.4)
    rows = _between(rng, 1, max(1, min(32768, 16384 * 4096 // cols)))
    case = {"op": op, "rows": rows, "cols": cols, "dtype": dt}
    if op != "keep":
        case["residual"] = rng.choice(["", dt, "fp32"])
        case["rms"] = rng.random() < 0.6
    return case


# ---------------------------------------------------------------------------
# what a program holds before the call
# ---------------------------------------------------------------------------
class _Maker:
    """Seeded inputs on the GPU; large ones in pieces, so that no full-size fp32 copy exists beside them."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(self, shape, dtype, std=1.0, mean=0.0):
        out = torch.empty(shape, dtype=dtype, device="cuda")
        flat, step = out.view(-1), 1 << 26
        for o in range(0, flat.numel(), step):
            part = flat[o:o + step]
            part.copy_(torch.randn(part.numel(), generator=self.gen, device="cuda") * std + mean)
        return out

    def uniform(self, shape, dtype, low, high):
        return (torch.rand(shape, generator=self.gen, device="cuda") * (high - low) + low).to(dtype)

    def logits(self, rows, cols, dtype):
        """A model's logits: spread 2.5 about a level, and per row a few tokens that stand out."""
        x = self.normal((rows, cols), dtype, 2.5, -3.0)
        best = torch.randint(0, cols, (rows, 3), generator=self.gen, device="cuda")
        high = torch.randn((rows, 3), generator=self.gen, device="cuda") * 2.0 + 8.0
        return x.scatter_(1, best, high.to(dtype)), best

    def tokens(self, best, cols, ignored):
        """Half of the rows name a token that stands out, half any; `ignored` rows are not scored."""
        rows = best.shape[0]
        anything = torch.randint(0, cols, (rows,), generator=self.gen, device="cuda")
        tok = torch.where(torch.rand(rows, generator=self.gen, device="cuda") < 0.5, best[:, 0], anything)
        tok[torch.randperm(rows, generator=self.gen, device="cuda")[:ignored]] = IGNORED
        return tok


def _pieces(rows, cols):
    step = max(1, _PIECE // max(cols, 1))
    return [(r, min(rows, r + step)) for r in range(0, rows, step)]


def _blocks(cols):
    return (cols + BLOCK - 1) // BLOCK


def _inputs(case, seed):
    """The seeded inputs alone, the same for every way of computing."""
    m, op, dt = _Maker(seed), case["op"], TYPES[case["dtype"]]
    rows, cols = case["rows"], case["cols"]
    s = {"op": op, "rows": rows, "cols": cols}
    if op in ("score", "grad"):
        s["x"], best = m.logits(rows, cols, dt)
        s["tokens"] = m.tokens(best, cols, case["ignored"])
        s["top"] = case.get("top", 0)
        if op == "grad":
            s["g"] = m.normal((rows,), torch.float32)
            s["h"] = m.normal((rows,), torch.float32, 0.01) if case["entropy"] else None
    elif op == "shard":
        # this rank holds the last but one shard; of the others, what they have sent: statistics and alternatives
        ranks, top = case["ranks"], case["top"]
        me = ranks - 2
        s.update(top=top, me=me, start=me * cols)
        s["stats"] = torch.zeros((ranks, 4, rows), dtype=torch.float32, device="cuda")
        s["top_value"] = torch.zeros((ranks, rows, top), dtype=torch.float32, device="cuda")
        s["top_token"] = torch.zeros((ranks, rows, top), dtype=torch.int64, device="cuda")
        firsts = []
        for r in range(ranks):
            x, best = m.logits(rows, cols, dt)
            firsts.append(best[:, 0] + r * cols)
            if r == me:
                s["x"] = x
            else:
                s.setdefault("others", {})[r] = x
        owner = torch.randint(0, ranks, (rows,), generator=m.gen, device="cuda")
        s["tokens"] = m.tokens(torch.stack(firsts, 1).gather(1, owner[:, None]), ranks * cols, case["ignored"])
    elif op == "keep":
        s["x"] = m.normal((rows, cols), dt) * m.uniform((rows, 1), dt, 0.1, 4.0)
    else:
        s["rms"] = case["rms"]
        rt = TYPES[case["residual"]] if case["residual"] else None
        s["gamma"] = m.uniform((cols,), dt, 0.8, 1.2)
        s["beta"] = None if case["rms"] else m.normal((cols,), dt, 0.1)
        x = m.normal((rows, cols), dt)
        if op == "norm":
            s["x"] = x
            s["residual"] = m.normal((rows, cols), rt, 2.0) if rt else None
        else:
            s["dz"] = m.normal((rows, cols), dt)
            s["dx_in"] = m.normal((rows, cols), rt) if rt else None
            s["rtype"] = rt
            # what the forward pass has left: the input in 8 bits, its statistics
            nb = _blocks(cols)
            s["q"] = torch.empty((rows, nb * BLOCK), dtype=torch.int8, device="cuda")
            s["scale"] = torch.empty((rows, nb), dtype=torch.uint8, device="cuda")
            s["mu"] = torch.empty(rows, device="cuda")
            s["rs"] = torch.empty(rows, device="cuda")
            for a, b in _pieces(rows, cols):
                f = x[a:b].float()
                s["q"][a:b], s["scale"][a:b] = _pack(f)
                s["mu"][a:b], s["rs"][a:b] = _moments(f, case["rms"])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    op, rows, cols = s["op"], s["rows"], s["cols"]
    f32 = {"dtype": torch.float32, "device": "cuda"}
    if op == "shard":
        for r, x in s.pop("others").items():
            for a, b in _pieces(rows, cols):
                st, tv, tt = _shard(x[a:b].float(), s["tokens"][a:b], r * cols, s["top"])
                s["stats"][r, :, a:b], s["top_value"][r, a:b], s["top_token"][r, a:b] = st, tv, tt
    if op == "grad":
        s["lse"], s["entropy"] = torch.empty(rows, **f32), torch.empty(rows, **f32)
        for a, b in _pieces(rows, cols):   # the forward pass's
            st, _, _ = _shard(s["x"][a:b].float(), s["tokens"][a:b], 0, 0)
            _, s["entropy"][a:b], s["lse"][a:b] = _merge(st[None], s["tokens"][a:b])
    # outputs that the program keeps from step to step
    if op in ("score", "shard"):
        s["logprob"], s["entropy"], s["lse"] = (torch.empty(rows, **f32) for _ in range(3))
        s["out_value"] = torch.empty((rows, s["top"]), **f32)
        s["out_token"] = torch.empty((rows, s["top"]), dtype=torch.int64, device="cuda")
    elif op == "grad":
        s["dx"] = torch.empty_like(s["x"])
    else:
        nb = _blocks(cols)
        src = s["x"] if "x" in s else s["dz"]
        if op != "norm_grad":
            s["q"] = torch.empty((rows, nb * BLOCK), dtype=torch.int8, device="cuda")
            s["scale"] = torch.empty((rows, nb), dtype=torch.uint8, device="cuda")
            s["kept"] = torch.empty((rows, cols), dtype=src.dtype, device="cuda")
        if op == "norm":
            s["z"] = torch.empty_like(src)
            s["sum"] = None if s["residual"] is None else torch.empty_like(s["residual"])
            s["mu"], s["rs"] = torch.empty(rows, **f32), torch.empty(rows, **f32)
        elif op == "norm_grad":
            s["z"], s["dx"] = torch.empty_like(src), torch.empty_like(src)
            s["dres"] = None if s["rtype"] is None else torch.empty((rows, cols), dtype=s["rtype"], device="cuda")
            s["dgamma"] = torch.empty_like(s["gamma"])
            s["dbeta"] = None if s["rms"] else torch.empty_like(s["gamma"])
    if own:
        hk = importlib.import_module("hotspa-ae_amd")
        s["hk"] = hk
        if op in ("score", "shard"):
            s["ws"] = _floats(hk.token_logprob_workspace_bytes(hk.dtype_code(s["x"]), rows, cols, s["top"]))
        elif op == "norm_grad":
            s["ws"] = _floats(hk.add_ln_q8_bwd_workspace_bytes(rows, cols))
    return s


def _floats(nbytes):
    """The workspace a program keeps for a call that asks for `nbytes` of it."""
    return torch.empty(max(1, (nbytes + 3) // 4), dtype=torch.float32, device="cuda")


# ---------------------------------------------------------------------------
# the plain form: elementary operations in 32 bits
# ---------------------------------------------------------------------------
def _shard(x, tokens, start, top):
    """(maximum, sum of exponentials, their first moment, picked logit) of the rows of one shard, [4, rows], and its
    `top` largest logits with their token numbers, ties to the lowest."""
    cols = x.shape[1]
    m = x.amax(1)
    d = x - m[:, None]
    e = torch.exp(d)
    s = e.sum(1)
    w = (e * d).sum(1)
    local = tokens - start
    inside = (local >= 0) & (local < cols)
    picked = torch.where(inside, x.gather(1, local.clamp(0, cols - 1)[:, None])[:, 0], torch.zeros_like(m))
    live = tokens != IGNORED
    stats = torch.stack([torch.where(live, m, torch.full_like(m, -math.inf))] +
                        [torch.where(live, v, torch.zeros_like(m)) for v in (s, w, picked)])
    values, numbers = _largest(x, torch.arange(cols, device=x.device).expand_as(x), top)
    return stats, values, numbers + start


def _largest(x, number, top):
    """The `top` largest of each row with their numbers, one after the other; of equal ones the lowest number."""
    values = torch.full((x.shape[0], top), -math.inf, dtype=x.dtype, device=x.device)
    numbers = torch.full((x.shape[0], top), -1, dtype=torch.int64, device=x.device)
    if top:
        x = x.clone()
    for k in range(min(top, x.shape[1])):
        v = x.amax(1, keepdim=True)
        n = torch.where(x == v, number, number.max() + 1).amin(1, keepdim=True)
        values[:, k], numbers[:, k] = v[:, 0], n[:, 0]
        x.masked_fill_(number == n, -math.inf)
    return values, numbers


def _merge(stats, tokens):
    """(log probability, entropy, log of the sum of exponentials) of the rows from the statistics [shards, 4, rows]."""
    m, s, w, picked = stats.unbind(1)
    top = m.amax(0)
    f = torch.where(s > 0, torch.exp(m - top), torch.zeros_like(s))
    d = torch.where(s > 0, m - top, torch.zeros_like(s))
    total = (s * f).sum(0)
    moment = (f * (w + d * s)).sum(0)
    log_s = torch.log(total)
    live = tokens != IGNORED
    zero = torch.zeros_like(top)
    return (torch.where(live, (picked.sum(0) - top) - log_s, zero), torch.where(live, log_s - moment / total, zero),
            torch.where(live, top + log_s, zero))


def _gradient(x, tokens, lse, entropy, g, h):
    live = tokens != IGNORED
    log_p = x - lse[:, None]
    p = torch.exp(log_p)
    out = -p * g[:, None]
    if h is not None:
        out -= p * (log_p + entropy[:, None]) * h[:, None]
    out += torch.where(torch.arange(x.shape[1], device=x.device)[None, :] == tokens[:, None], g[:, None],
                       torch.zeros_like(g)[:, None])
    return torch.where(live[:, None], out, torch.zeros_like(out))


def _pack(x):
    """fp32 rows -> (int8 [rows, blocks * 32], exponents uint8 [rows, blocks])."""
    rows, cols = x.shape
    nb = _blocks(cols)
    padded = torch.zeros((rows, nb * BLOCK), dtype=torch.float32, device=x.device)
    padded[:, :cols] = x
    b = padded.view(rows, nb, BLOCK)
    e = ((b.abs().amax(2).contiguous().view(torch.int32) >> 23) & 255).clamp(min=7)
    factor = ((260 - e) << 23).view(torch.float32)                      # 2^(133 - e)
    q = torch.round(b * factor[:, :, None]).clamp(-127, 127).to(torch.int8)
    return q.view(rows, nb * BLOCK), e.to(torch.uint8)


def _unpack(q, scale, cols):
    rows, nb = scale.shape
    factor = torch.exp2(scale.double() - 133.0).float()
    return (q.view(rows, nb, BLOCK).float() * factor[:, :, None]).view(rows, nb * BLOCK)[:, :cols]


def _moments(x, rms):
    mu = x.mean(1)
    if rms:
        return mu, 1.0 / torch.sqrt((x * x).mean(1) + EPS)
    d = x - mu[:, None]
    return mu, 1.0 / torch.sqrt((d * d).mean(1) + EPS)


def _affine(x, mu, rs, gamma, beta, rms):
    n = (x if rms else x - mu[:, None]) * rs[:, None]
    return n * gamma.float() if beta is None else n * gamma.float() + beta.float()


def _norm_gradient(dz, x, mu, rs, gamma, dx_in, rms):
    """(gradient of the input, parts of gamma's and beta's gradients) of some rows."""
    n = (x if rms else x - mu[:, None]) * rs[:, None]
    t = dz * gamma.float()
    dx = t - n * (t * n).mean(1, keepdim=True)
    if not rms:
        dx = dx - t.mean(1, keepdim=True)
    dx = dx * rs[:, None]
    if dx_in is not None:
        dx = dx + dx_in.float()
    return dx, (dz * n).sum(0, dtype=torch.float64), dz.sum(0, dtype=torch.float64)


def _run_plain(s):
    op, rows, cols = s["op"], s["rows"], s["cols"]
    parts = _pieces(rows, cols)
    if op == "score":
        for a, b in parts:
            st, tv, tt = _shard(s["x"][a:b].float(), s["tokens"][a:b], 0, s["top"])
            s["logprob"][a:b], s["entropy"][a:b], s["lse"][a:b] = _merge(st[None], s["tokens"][a:b])
            s["out_value"][a:b], s["out_token"][a:b] = tv - s["lse"][a:b, None], tt
        return [s[k] for k in ("logprob", "entropy", "lse", "out_value", "out_token")]
    if op == "shard":
        me = s["me"]
        for a, b in parts:
            st, tv, tt = _shard(s["x"][a:b].float(), s["tokens"][a:b], s["start"], s["top"])
            s["stats"][me, :, a:b], s["top_value"][me, a:b], s["top_token"][me, a:b] = st, tv, tt
        lp, ent, lse = _merge(s["stats"], s["tokens"])
        # shards follow each other, so that of equal values the first is the one with the lowest number
        v = s["top_value"].permute(1, 0, 2).reshape(rows, -1)
        n = s["top_token"].permute(1, 0, 2).reshape(rows, -1)
        values, numbers = _largest(v, n, s["top"])
        return [lp, ent, lse, values - lse[:, None], numbers]
    if op == "grad":
        for a, b in parts:
            s["dx"][a:b] = _gradient(s["x"][a:b].float(), s["tokens"][a:b], s["lse"][a:b], s["entropy"][a:b],
                                     s["g"][a:b], None if s["h"] is None else s["h"][a:b])
        return [s["dx"]]
    if op == "keep":
        for a, b in parts:
            s["q"][a:b], s["scale"][a:b] = _pack(s["x"][a:b].float())
            s["kept"][a:b] = _unpack(s["q"][a:b], s["scale"][a:b], cols)
        return [s["kept"]]
    if op == "norm":
        for a, b in parts:
            x = s["x"][a:b].float()
            if s["residual"] is not None:
                x = x + s["residual"][a:b].float()
                s["sum"][a:b] = x
            s["q"][a:b], s["scale"][a:b] = _pack(x)
            s["mu"][a:b], s["rs"][a:b] = _moments(x, s["rms"])
            s["z"][a:b] = _affine(x, s["mu"][a:b], s["rs"][a:b], s["gamma"], s["beta"], s["rms"])
            s["kept"][a:b] = _unpack(s["q"][a:b], s["scale"][a:b], cols)
        return [s[k] for k in ("z", "sum", "mu", "rs", "kept") if s[k] is not None]
    dgamma = dbeta = 0.0
    for a, b in parts:
        x = _unpack(s["q"][a:b], s["scale"][a:b], cols)
        mu, rs = s["mu"][a:b], s["rs"][a:b]
        s["z"][a:b] = _affine(x, mu, rs, s["gamma"], s["beta"], s["rms"])
        dx, dg, db = _norm_gradient(s["dz"][a:b].float(), x, mu, rs, s["gamma"],
                                    None if s["dx_in"] is None else s["dx_in"][a:b], s["rms"])
        s["dx"][a:b] = dx
        if s["dres"] is not None:
            s["dres"][a:b] = dx
        dgamma, dbeta = dgamma + dg, dbeta + db
    s["dgamma"].copy_(dgamma)
    if s["dbeta"] is not None:
        s["dbeta"].copy_(dbeta)
    return [s[k] for k in ("z", "dx", "dres", "dgamma", "dbeta") if s[k] is not None]


def _run_own(s):
    hk, op = s["hk"], s["op"]
    if op == "score":
        hk.token_logprob_fwd(s["x"], s["tokens"], s["logprob"], s["entropy"], s["lse"], s["out_value"], s["out_token"],
                             IGNORED, workspace=s["ws"])
        return [s[k] for k in ("logprob", "entropy", "lse", "out_value", "out_token")]
    if op == "shard":
        me = s["me"]
        hk.vocab_parallel_logprob_stats(s["x"], s["tokens"], s["stats"][me], s["top_value"][me], s["top_token"][me],
                                        s["start"], IGNORED, workspace=s["ws"])
        hk.vocab_parallel_logprob_combine(s["stats"], s["top_value"], s["top_token"], s["tokens"], IGNORED, s["logprob"],
                                          s["entropy"], s["lse"], s["out_value"], s["out_token"])
        return [s[k] for k in ("logprob", "entropy", "lse", "out_value", "out_token")]
    if op == "grad":
        hk.token_logprob_bwd(s["x"], s["tokens"], s["lse"], s["entropy"], s["g"], s["h"], s["dx"], IGNORED)
        return [s["dx"]]
    if op == "keep":
        hk.q8_pack(s["x"], s["q"], s["scale"])
        hk.q8_unpack(s["q"], s["scale"], s["kept"])
        return [s["kept"]]
    if op == "norm":
        hk.add_ln_q8_fwd(s["x"], s["residual"], s["gamma"], s["beta"], s["z"], s["sum"], s["q"], s["scale"], s["mu"],
                         s["rs"], EPS, s["rms"])
        hk.q8_unpack(s["q"], s["scale"], s["kept"])
        return [s[k] for k in ("z", "sum", "mu", "rs", "kept") if s[k] is not None]
    hk.add_ln_q8_out(s["q"], s["scale"], s["mu"], s["rs"], s["gamma"], s["beta"], s["z"], s["rms"])
    hk.add_ln_q8_bwd(s["dz"], s["dx_in"], s["q"], s["scale"], s["mu"], s["rs"], s["gamma"], s["dx"], s["dres"],
                     s["dgamma"], s["dbeta"], s["rms"], workspace=s["ws"])
    return [s[k] for k in ("z", "dx", "dres", "dgamma", "dbeta") if s[k] is not None]


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    """Bytes and operations of one pass: every input read once, every output written once (the 8 bits too, which the
    passes of "keep" and "norm" read back to hand out the values they stand for)."""
    rows, cols, op, es = case["rows"], case["cols"], case["op"], SIZE[case["dtype"]]
    live = rows - case.get("ignored", 0)
    n, kept = rows * cols, rows * _blocks(cols) * (BLOCK + 1)
    if op == "score":
        return {"bytes": live * cols * es + rows * (8 + 12 + 12 * case["top"]), "flops": 6 * live * cols}
    if op == "shard":
        return {"bytes": live * cols * es + rows * (8 + 12 + 12 * case["top"]) +
                case["ranks"] * rows * (16 + 12 * case["top"]), "flops": 6 * live * cols}
    if op == "grad":
        return {"bytes": (live + rows) * cols * es + rows * (8 + 12 + 4 * case["entropy"]),
                "flops": (8 if case["entropy"] else 4) * live * cols}
    if op == "keep":
        return {"bytes": 2 * n * es + kept, "flops": 4 * n}
    rs = SIZE[case["residual"]] if case["residual"] else 0
    params = cols * es * (1 if case["rms"] else 2)
    if op == "norm":
        return {"bytes": n * (3 * es + 2 * rs) + kept + params + 8 * rows, "flops": 10 * n}
    return {"bytes": n * (3 * es + 2 * rs) + kept + 3 * params + 8 * rows, "flops": 16 * n}


# ---------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------
def _exact_scores(x, tokens):
    """(log probability, entropy, log of the sum of exponentials) of whole rows."""
    lse = torch.logsumexp(x, 1)
    lp = x - lse[:, None]
    picked = lp.gather(1, tokens.clamp(min=0)[:, None])[:, 0]
    entropy = -(torch.exp(lp) * lp).sum(1)
    gone = tokens == IGNORED
    return tuple(v.masked_fill(gone, 0.0) for v in (picked, entropy, lse))


def _exact_top(x, top):
    """Values and columns of the `top` largest, by sorting."""
    values, order = torch.sort(x, dim=1, descending=True, stable=True)
    return values[:, :top], order[:, :top]


def _power_of_two(n):
    """2^n as fp64, from its bits: a power function may be off in the last place, which moves values at a border."""
    return ((n + 1023) << 52).view(torch.float64)


def exact(case, seed):
    s = _inputs(case, seed)
    op, rows, cols = s["op"], s["rows"], s["cols"]
    outs = []

    def gather(parts):
        outs.append(parts)

    step = max(1, (1 << 26) // (cols * case.get("ranks", 1)))
    for a in range(0, rows, step):
        b = min(rows, a + step)
        if op in ("score", "shard"):
            if op == "shard":
                x = torch.cat([s["x"][a:b] if r == s["me"] else s["others"][r][a:b] for r in range(case["ranks"])], 1)
            else:
                x = s["x"][a:b]
            x = x.double()
            picked, entropy, lse = _exact_scores(x, s["tokens"][a:b])
            values, order = _exact_top(x, s["top"])
            gather([picked, entropy, lse, values - lse[:, None], order])
        elif op == "grad":
            x = s["x"][a:b].double()
            tok = s["tokens"][a:b]
            lp = torch.log_softmax(x, 1)
            p = torch.exp(lp)
            one = torch.nn.functional.one_hot(tok.clamp(min=0), cols)
            dx = s["g"][a:b, None].double() * (one - p)
            if s["h"] is not None:
                mean = (p * lp).sum(1, keepdim=True)
                dx -= s["h"][a:b, None].double() * p * (lp - mean)
            gather([dx.masked_fill((tok == IGNORED)[:, None], 0.0)])
        elif op in ("keep", "norm"):
            x = s["x"][a:b].float()
            if op == "norm" and s["residual"] is not None:
                x = x + s["residual"][a:b].float()          # what is normalised and kept is this sum in fp32
            x = x.double()
            pad = torch.nn.functional.pad(x, (0, -cols % BLOCK)).view(b - a, -1, BLOCK)
            _, power = torch.frexp(pad.abs().amax(2, keepdim=True))   # 2^(power - 1) <= largest < 2^power
            unit = _power_of_two((power.long() - 1).clamp(min=-120) - 6)
            kept = ((pad / unit).round().clamp(-127, 127) * unit).view(b - a, -1)[:, :cols]
            if op == "keep":
                gather([kept])
                continue
            mu = x.mean(1)
            spread = (x * x).mean(1) if s["rms"] else x.var(1, correction=0)
            rs = (spread + EPS) ** -0.5
            z = (x if s["rms"] else x - mu[:, None]) * rs[:, None] * s["gamma"].double()
            if s["beta"] is not None:
                z = z + s["beta"].double()
            gather([z] + ([x] if s["residual"] is not None else []) + [mu, rs, kept])
        else:
            unit = _power_of_two(s["scale"][a:b].long() - 133)
            x = (s["q"][a:b].double().view(b - a, -1, BLOCK) * unit[:, :, None]).view(b - a, -1)[:, :cols]
            rs = s["rs"][a:b, None].double()
            n = (x if s["rms"] else x - s["mu"][a:b, None].double()) * rs
            dz, gamma = s["dz"][a:b].double(), s["gamma"].double()
            z = gamma * n + (0.0 if s["beta"] is None else s["beta"].double())
            dn = dz * gamma
            back = dn - n * (dn * n).sum(1, keepdim=True) / cols
            if not s["rms"]:
                back = back - dn.sum(1, keepdim=True) / cols
            dx = back * rs + (0.0 if s["dx_in"] is None else s["dx_in"][a:b].double())
            gather([z, dx] + ([dx] if s["rtype"] else []) + [(dz * n).sum(0)] + ([] if s["rms"] else [dz.sum(0)]))
    if op == "norm_grad":
        sums = 1 if s["rms"] else 2
        whole = [torch.cat(c) for c in list(zip(*outs))[:-sums]]
        return whole + [torch.stack(c).sum(0) for c in list(zip(*outs))[-sums:]]
    return [torch.cat(c) for c in zip(*outs)]
