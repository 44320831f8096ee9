"""Four operators of a language model's training step, as a program built on
this library runs them through the C entry points of include/mle_hip.h.

A case is a dict of plain values; `kind` names the operator and the rest are its
sizes and options:

  xent       the vocabulary's output projection with its cross entropy, in
             pieces of the vocabulary: forward (loss, row losses, row
             log-sums), then dX, dW and db; no logits are kept
  q8_linear  activations kept in 8 bits for the backward pass: a Linear's
             input, quantised in the forward, and its weight and bias gradient
  q8_act     the same for an activation function's input: forward and backward
  norm       the residual Add and the root-mean-square norm that reads it, with
             the output also in 8 bits: forward, reading the 8 bits back, and
             backward
  embed      embedding lookup with scaling, and the table's gradient by sorted
             tokens

Tensors are float32 and token ids int32.  8-bit tensors are signed codes with
one power-of-two scale per 32 consecutive values of a row: the smallest 2^k,
k >= -126, for which the largest magnitude stays below 127.5 steps of it.
Gradients are assigned, as in a step after zero_grad.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
EPS = 1e-5       # the norm's epsilon
GROUP = 32       # values that share a scale
MAX_FLOPS = 1.62e12  # of a drawn case: the largest listed one's
MAX_BYTES = 2.9e9

# --------------------------------------------------------------------- cases


def listed() -> list[dict]:
    return [
        # A short batch of a small model: latency.
        dict(name="xent_small", kind="xent", rows=64, d=256, vocab=4096, bias=1, ignored=0),
        # The transformer block's vocabulary projection and loss (32 x 256 tokens).
        dict(name="xent_block", kind="xent", rows=8192, d=512, vocab=8000, bias=1, ignored=0),
        # Padded sequences of no round size, some of whose tokens take no part.
        dict(name="xent_ragged", kind="xent", rows=1000, d=330, vocab=10007, bias=1, ignored=1),
        # A large vocabulary: the logits alone would be 1 GB.
        dict(name="xent_large", kind="xent", rows=8192, d=1024, vocab=32000, bias=0, ignored=1),
        # The benchmark's Linear at its full width.
        dict(name="q8_linear_wide", kind="q8_linear", rows=8192, inp=1024, out=4096),
        # A small Linear on a short batch, no size a multiple of a tile.
        dict(name="q8_linear_ragged", kind="q8_linear", rows=1000, inp=330, out=516),
        # The transformer block's feed-forward activation.
        dict(name="q8_act_block", kind="q8_act", rows=8192, cols=2048, act="gelu"),
        # One short sequence: latency.
        dict(name="norm_small", kind="norm", rows=64, cols=256, residual=1),
        # The transformer block's residual stream.
        dict(name="norm_block", kind="norm", rows=8192, cols=512, residual=1),
        # A wide model's residual stream.
        dict(name="norm_wide", kind="norm", rows=16384, cols=4096, residual=1),
        # The transformer block's tokens.
        dict(name="embed_block", kind="embed", batch=32, clen=256, max_clen=256, vocab=8000, dim=512),
        # A large vocabulary and padded sequences; frequent tokens have
        # thousands of places.
        dict(name="embed_large", kind="embed", batch=16, clen=2000, max_clen=2048, vocab=128000, dim=1024),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng: random.Random, lo: int, hi: int) -> int:
    """A layer width: mostly a multiple of 16, sometimes of 4, sometimes any."""
    w = _log_int(rng, lo, hi)
    m = rng.choice((16, 16, 4, 1))
    return max(m, w // m * m)


def _draw_once(rng: random.Random) -> dict:
    kind = rng.choice(("xent", "xent", "xent", "q8_linear", "q8_linear", "q8_act", "norm", "norm", "embed", "embed"))
    if kind == "xent":
        return dict(kind=kind, rows=_log_int(rng, 32, 8192), d=_width(rng, 64, 1024), vocab=_width(rng, 256, 32000),
                    bias=rng.randint(0, 1), ignored=rng.randint(0, 1))
    if kind == "q8_linear":
        return dict(kind=kind, rows=_log_int(rng, 64, 16384), inp=_width(rng, 48, 4096), out=_width(rng, 48, 4096))
    if kind == "q8_act":
        return dict(kind=kind, rows=_log_int(rng, 16, 16384), cols=_width(rng, 48, 4096),
                    act=rng.choice(("relu", "gelu", "silu")))
    if kind == "norm":
        return dict(kind=kind, rows=_log_int(rng, 16, 16384), cols=_width(rng, 64, 8192), residual=rng.randint(0, 1))
    clen = _log_int(rng, 16, 2048)
    return dict(kind=kind, batch=_log_int(rng, 1, 32), clen=clen, max_clen=clen + rng.choice((0, 0, rng.randint(1, 64))),
                vocab=_log_int(rng, 256, 128000), dim=_width(rng, 48, 1024))


def draw(rng: random.Random) -> dict:
    while True:
        case = _draw_once(rng)
        w = work(case)
        if w["flops"] <= MAX_FLOPS and w["bytes"] <= MAX_BYTES:
            return case


def work(case: dict) -> dict:
    c, k = case, case["kind"]
    if k == "xent":
        r, d, v = c["rows"], c["d"], c["vocab"]
        # X, W, ids and bias read; loss, row losses, log-sums, dX, dW, db written
        return dict(flops=6.0 * r * d * v, bytes=4.0 * (2 * r * d + 2 * d * v + v * (1 + c["bias"]) + 3 * r))
    if k == "q8_linear":
        r, i, o = c["rows"], c["inp"], c["out"]
        # x read, its 8 bits written and read; dY read; dW and db written
        return dict(flops=2.0 * r * i * o, bytes=r * i * (4.0 + 2 * (1 + 1 / GROUP)) + 4.0 * (r * o + i * o + o))
    if k == "q8_act":
        # x read; y and the 8 bits written; the 8 bits and dy read; dx written
        return dict(flops=0.0, bytes=c["rows"] * c["cols"] * (16.0 + 2 * (1 + 1 / GROUP)))
    if k == "norm":
        n = c["rows"] * c["cols"]
        # x, the residual, dy and dres read; h, y, the 8 bits, their values and
        # dh written; h and the 8 bits read again
        return dict(flops=0.0, bytes=n * (4.0 * (8 + 2 * c["residual"]) + 2 * (1 + 1 / GROUP)) + 8.0 * c["cols"])
    n = c["batch"] * c["clen"]
    # the rows that the tokens name are read, at most the whole table; the
    # output and the whole gradient are written
    return dict(flops=0.0, bytes=4.0 * (c["dim"] * (2 * n + min(n, c["vocab"]) + c["vocab"]) + 2 * n))


# ------------------------------------------------------------------- prepare


def _normal(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV).mul_(scale)


def _uniform(g, *shape, bound=1.0):
    return torch.rand(*shape, generator=g, device=DEV).mul_(2 * bound).sub_(bound)


def _frequent(g, n, vocab):
    """Token ids as text has them: id k about 1 / (k + 1) as often as id 0."""
    u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
    return torch.exp(u * math.log(vocab + 1.0)).long().sub_(1).clamp_(0, vocab - 1).to(torch.int32)


def _new(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device=DEV)


def _ws(nbytes):
    return _new(max(int(nbytes), 16), dtype=torch.uint8)


def _groups(cols):
    return -(-cols // GROUP)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = _PREPARE[case["kind"]](case, g)
    s["case"] = case
    return s


def _prep_xent(c, g):
    r, d, v = c["rows"], c["d"], c["vocab"]
    # weights of a trained projection, and rows that lean towards their target:
    # logits of order one, targets well above the mean
    w = _uniform(g, d, v, bound=math.sqrt(3.0 / d))
    keys = _frequent(g, r, v)
    lean = torch.rand(r, 1, generator=g, device=DEV) * 6.0
    x = _normal(g, r, d) + lean * w[:, keys.long()].t()
    if c["ignored"]:
        keys[torch.rand(r, generator=g, device=DEV) < 0.15] = -1
    taken = max(1, int((keys >= 0).sum()))
    s = dict(x=x, w=w, b=_uniform(g, v, bound=0.5) if c["bias"] else None, keys=keys, scale=1.0 / taken)
    if own:
        from ml_engine_amd import hip
        hip.init(0)
        s.update(loss=_new(1), row_loss=_new(r), lse=_new(r), dx=_new(r, d), dw=_new(d, v), db=_new(v),
                 ws=_ws(hip.lib().mle_vocab_xent_ws_bytes(r, d, v)))
    return s


def _prep_q8_linear(c, g):
    r, i, o = c["rows"], c["inp"], c["out"]
    # a feed-forward's inner activations, some channels of which are large
    x = torch.relu(_normal(g, r, i)) + _normal(g, r, i, scale=0.1)
    x *= 1.0 + 9.0 * (torch.rand(i, generator=g, device=DEV) < 0.02)
    s = dict(x=x, dy=_normal(g, r, o, scale=1e-3))
    if own:
        from ml_engine_amd import hip
        hip.init(0)
        s.update(q=_new(r, i, dtype=torch.int8), e=_new(r, _groups(i), dtype=torch.uint8), dw=_new(i, o), db=_new(o),
                 ws=_ws(hip.lib().mle_q8_linear_wgrad_ws_bytes(r, i, o)))
    return s


def _prep_q8_act(c, g):
    r, n = c["rows"], c["cols"]
    s = dict(x=_normal(g, r, n, scale=1.5), dy=_normal(g, r, n, scale=1e-3))
    if own:
        from ml_engine_amd import hip
        hip.init(0)
        s.update(q=_new(r, n, dtype=torch.int8), e=_new(r, _groups(n), dtype=torch.uint8), y=_new(r, n), dx=_new(r, n))
    return s


def _prep_norm(c, g):
    r, n = c["rows"], c["cols"]
    s = dict(x=_normal(g, r, n, scale=0.5), r=_normal(g, r, n) if c["residual"] else None,
             w=1.0 + _normal(g, n, scale=0.1), dy=_normal(g, r, n, scale=1e-3),
             dres=_normal(g, r, n, scale=1e-3) if c["residual"] else None)
    if own:
        from ml_engine_amd import hip
        hip.init(0)
        s.update(h=_new(r, n), y=_new(r, n), rstd=_new(r), q=_new(r, n, dtype=torch.int8),
                 e=_new(r, _groups(n), dtype=torch.uint8), back=_new(r, n), dh=_new(r, n), dw=_new(n),
                 ws=_ws(hip.lib().mle_add_rmsnorm_ws_bytes(r, n)))
    return s


def _prep_embed(c, g):
    b, n, m, v, d = c["batch"], c["clen"], c["max_clen"], c["vocab"], c["dim"]
    keys = _frequent(g, b * m, v).view(b, m)
    keys[:, n:] = -1                                # past the longest sequence
    ends = torch.randint(n // 2, n + 1, (b, 1), generator=g, device=DEV)
    keys[torch.arange(m, device=DEV)[None, :] >= ends] = -1  # past each one's own
    s = dict(keys=keys, table=_normal(g, v, d, scale=d ** -0.5), dy=_normal(g, b, n, d, scale=1e-3),
             scale=math.sqrt(d))
    if own:
        from ml_engine_amd import hip
        hip.init(0)
        L = hip.lib()
        s.update(out=_new(b, n, d), dtable=_new(v, d), index=_ws(L.mle_embed_sorted_index_bytes(b, n, v)),
                 ws=_ws(L.mle_embed_sorted_grad_ws_bytes(b, n, d)))
    return s


_PREPARE = dict(xent=_prep_xent, q8_linear=_prep_q8_linear, q8_act=_prep_q8_act, norm=_prep_norm, embed=_prep_embed)

# ----------------------------------------------------------------------- run


def run(state: dict):
    k = state["case"]["kind"]
    return _OWN[k](state, state["case"]) if own else _PLAIN[k](state, state["case"])


def _p(t):
    return None if t is None else t.data_ptr()


def _own_xent(s, c):
    from ml_engine_amd import hip
    r, d, v = c["rows"], c["d"], c["vocab"]
    hip.call("mle_vocab_xent_fwd", None, r, d, v, _p(s["x"]), d, _p(s["w"]), v, _p(s["b"]), _p(s["keys"]), r, r,
             s["scale"], _p(s["lse"]), _p(s["row_loss"]), _p(s["loss"]), _p(s["ws"]), s["ws"].numel())
    hip.call("mle_vocab_xent_bwd", None, r, d, v, _p(s["x"]), d, _p(s["w"]), v, _p(s["b"]), _p(s["keys"]), r, r,
             _p(s["lse"]), None, s["scale"], _p(s["dx"]), d, 0, _p(s["dw"]), v, _p(s["db"]), 0, _p(s["ws"]),
             s["ws"].numel())
    return {k: s[k] for k in ("loss", "row_loss", "lse", "dx", "dw", "db")}


def _own_q8_linear(s, c):
    from ml_engine_amd import hip
    r, i, o, ne = c["rows"], c["inp"], c["out"], s["e"].shape[1]
    hip.call("mle_q8_quantize", None, r, i, _p(s["x"]), i, _p(s["q"]), i, _p(s["e"]), ne)
    hip.call("mle_q8_linear_wgrad", None, r, i, o, _p(s["q"]), i, _p(s["e"]), ne, _p(s["dy"]), o, _p(s["dw"]), o,
             _p(s["db"]), 0, _p(s["ws"]), s["ws"].numel())
    return {k: s[k] for k in ("dw", "db")}


def _own_q8_act(s, c):
    from ml_engine_amd import hip
    r, n, ne, kind = c["rows"], c["cols"], s["e"].shape[1], hip.ACT[c["act"]]
    hip.call("mle_q8_act_fwd", None, kind, r, n, _p(s["x"]), n, _p(s["y"]), n, _p(s["q"]), n, _p(s["e"]), ne)
    hip.call("mle_q8_act_bwd", None, kind, r, n, _p(s["q"]), n, _p(s["e"]), ne, _p(s["dy"]), n, _p(s["dx"]), n, 0)
    return {k: s[k] for k in ("y", "dx")}


def _own_norm(s, c):
    from ml_engine_amd import hip
    r, n, ne = c["rows"], c["cols"], s["e"].shape[1]
    h = s["h"] if c["residual"] else s["x"]  # without a residual x is what the backward reads
    hip.call("mle_add_rmsnorm_q8_fwd", None, r, n, _p(s["x"]), _p(s["r"]), _p(s["w"]), EPS,
             _p(h) if c["residual"] else None, _p(s["y"]), _p(s["rstd"]), _p(s["q"]), n, _p(s["e"]), ne)
    hip.call("mle_q8_dequantize", None, r, n, _p(s["q"]), n, _p(s["e"]), ne, _p(s["back"]), n)
    hip.call("mle_add_rmsnorm_bwd", None, r, n, _p(h), _p(s["w"]), _p(s["rstd"]), _p(s["dy"]), _p(s["dres"]),
             _p(s["dh"]), 0, _p(s["dw"]), 0, _p(s["ws"]), s["ws"].numel())
    return dict(h=h, y=s["y"], back=s["back"], dh=s["dh"], dw=s["dw"])


def _own_embed(s, c):
    from ml_engine_amd import hip
    b, n, m, v, d = c["batch"], c["clen"], c["max_clen"], c["vocab"], c["dim"]
    hip.call("mle_embed_scaled_fwd", None, _p(s["out"]), _p(s["table"]), _p(s["keys"]), b, n, m, d, v, s["scale"],
             _p(s["index"]), s["index"].numel())
    hip.call("mle_embed_sorted_grad", None, _p(s["dtable"]), _p(s["dy"]), _p(s["index"]), s["index"].numel(), b, n, d, v,
             s["scale"], 0, _p(s["ws"]), s["ws"].numel())
    return {k: s[k] for k in ("out", "dtable")}


_OWN = dict(xent=_own_xent, q8_linear=_own_q8_linear, q8_act=_own_q8_act, norm=_own_norm, embed=_own_embed)

# ---------------------------------------------------------------- plain form


def _plain_xent(s, c):
    x, w, keys = s["x"], s["w"], s["keys"].long()
    rows = torch.arange(c["rows"], device=DEV)
    valid = keys >= 0
    at = keys.clamp(min=0)
    logits = x @ w
    if s["b"] is not None:
        logits += s["b"]
    top = logits.amax(1, keepdim=True)
    target = logits[rows, at]
    e = (logits - top).exp_()
    total = e.sum(1, keepdim=True)
    lse = (top + total.log()).squeeze(1)
    row_loss = torch.where(valid, lse - target, torch.zeros_like(lse))
    p = e.div_(total)
    p[rows, at] -= 1.0
    p *= (valid * s["scale"])[:, None]
    return dict(loss=(row_loss.sum() * s["scale"]).view(1), row_loss=row_loss, lse=lse, dx=p @ w.t(), dw=x.t() @ p,
                db=p.sum(0))


def _plain_q8(x):
    """The values that x's 8 bits stand for; in 64 bits, where every step is exact."""
    r, n = x.shape
    pad = _groups(n) * GROUP - n
    v = torch.nn.functional.pad(x.double(), (0, pad)).view(r, -1, GROUP)
    m, k = torch.frexp(v.abs().amax(2, keepdim=True))  # m 2^k, 1/2 <= m < 1
    k = (k - torch.where(m < 127.5 / 128, 7, 6)).clamp(min=-126)
    return torch.ldexp(torch.ldexp(v, -k).round(), k).view(r, -1)[:, :n].float()


def _plain_act(kind, x):
    if kind == "relu":
        return x.clamp(min=0)
    if kind == "silu":
        return x / (1 + (-x).exp())
    return 0.5 * x * (1 + (math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)).tanh())


def _plain_act_grad(kind, x):
    if kind == "relu":
        return (x > 0).float()
    if kind == "silu":
        sg = 1 / (1 + (-x).exp())
        return sg * (1 + x * (1 - sg))
    t = (math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)).tanh()
    return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * (math.sqrt(2 / math.pi) * (1 + 0.134145 * x * x))


def _plain_q8_linear(s, c):
    return dict(dw=_plain_q8(s["x"]).t() @ s["dy"], db=s["dy"].sum(0))


def _plain_q8_act(s, c):
    return dict(y=_plain_act(c["act"], s["x"]), dx=_plain_act_grad(c["act"], _plain_q8(s["x"])) * s["dy"])


def _plain_norm(s, c):
    h = s["x"] + s["r"] if c["residual"] else s["x"]
    # y in 64 bits and rounded once: its 8 bits turn on the last place of it
    h64 = h.double()
    rstd = 1.0 / (h64.square().mean(1, keepdim=True) + EPS).sqrt()
    y = (h64 * rstd * s["w"].double()).float()
    unit = h * rstd.float()
    gy = s["dy"] * s["w"]
    dh = rstd.float() * (gy - unit * (gy * unit).mean(1, keepdim=True))
    if s["dres"] is not None:
        dh = dh + s["dres"]
    return dict(h=h, y=y, back=_plain_q8(y), dh=dh, dw=(s["dy"] * unit).sum(0))


def _plain_embed(s, c):
    n, v, d = c["clen"], c["vocab"], c["dim"]
    keys = s["keys"][:, :n].reshape(-1).long()
    valid = keys >= 0
    out = s["table"][keys.clamp(min=0)] * (valid * s["scale"])[:, None]
    dtable = torch.zeros(v, d, device=DEV)
    dtable.index_add_(0, keys[valid], s["dy"].view(-1, d)[valid])
    return dict(out=out.view(-1, n, d), dtable=dtable * s["scale"])


_PLAIN = dict(xent=_plain_xent, q8_linear=_plain_q8_linear, q8_act=_plain_q8_act, norm=_plain_norm, embed=_plain_embed)

# --------------------------------------------------------------------- exact


def exact(case: dict, seed: int):
    """What run() returns for prepare(case, seed), in 64 bits."""
    s = prepare(case, seed)
    return _EXACT[case["kind"]](s, case)


def _exact_xent(s, c):
    x, w = s["x"].double(), s["w"].double()
    keep = torch.nonzero(s["keys"] >= 0).squeeze(1)
    keys = s["keys"][keep].long()
    logits = torch.matmul(x, w)
    if s["b"] is not None:
        logits = logits + s["b"].double()[None, :]
    lse = torch.logsumexp(logits, 1)
    row_loss = torch.zeros_like(lse)
    row_loss[keep] = lse[keep] - logits[keep].gather(1, keys[:, None]).squeeze(1)
    grad = torch.zeros_like(logits)
    grad[keep] = torch.exp(logits[keep] - lse[keep, None]) * s["scale"]
    del logits
    grad.index_put_((keep, keys), torch.full_like(lse[keep], -s["scale"]), accumulate=True)
    return dict(loss=row_loss.sum().view(1) * s["scale"], row_loss=row_loss, lse=lse, dx=torch.matmul(grad, w.t()),
                dw=torch.matmul(x.t(), grad), db=grad.sum(0))


def _exact_q8(x):
    """The nearest multiple of each group's step; the step is raised where the first guess is one too small."""
    r, n = x.shape
    at = torch.arange(n, device=DEV).div(GROUP, rounding_mode="floor").expand(r, n)
    top = torch.zeros(r, _groups(n), dtype=torch.float64, device=DEV).scatter_reduce_(1, at, x.abs().double(), "amax")
    step = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -149))) - 6)
    step = torch.where(top < 127.5 * step, step, 2 * step).clamp(min=2.0 ** -126).gather(1, at)
    return torch.round(x.double() / step) * step


def _exact_act(kind, x):
    if kind == "relu":
        return torch.relu(x)
    if kind == "silu":
        return x * torch.sigmoid(x)
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))


def _exact_q8_linear(s, c):
    dy = s["dy"].double()
    return dict(dw=torch.matmul(_exact_q8(s["x"]).t(), dy), db=dy.sum(0))


def _exact_q8_act(s, c):
    kept = _exact_q8(s["x"]).requires_grad_(True)
    slope, = torch.autograd.grad(_exact_act(c["act"], kept).sum(), kept)
    if c["act"] == "relu":
        slope = (kept.detach() > 0).double()
    return dict(y=_exact_act(c["act"], s["x"].double()), dx=slope * s["dy"].double())


def _exact_norm(s, c):
    # the sum is held in 32 bits, as is the output that the 8 bits are made of
    h = (s["x"].double() + s["r"].double()).float().double() if c["residual"] else s["x"].double()
    h.requires_grad_(True)
    w = s["w"].double().requires_grad_(True)
    y = w * h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
    dh, dw = torch.autograd.grad(y, (h, w), s["dy"].double())
    if s["dres"] is not None:
        dh = dh + s["dres"].double()
    y = y.detach()
    return dict(h=h.detach(), y=y, back=_exact_q8(y.float()), dh=dh, dw=dw)


def _exact_embed(s, c):
    n, v, d = c["clen"], c["vocab"], c["dim"]
    keys = s["keys"][:, :n].reshape(-1).long()
    keys = torch.where(keys < 0, v, keys)  # one row more, for the tokens that take no part
    table = torch.cat([s["table"].double(), torch.zeros(1, d, dtype=torch.float64, device=DEV)])
    out = (table * s["scale"]).index_select(0, keys)
    grad = torch.zeros(v + 1, d, dtype=torch.float64, device=DEV)
    grad.scatter_add_(0, keys[:, None].expand(-1, d), s["dy"].double().view(-1, d) * s["scale"])
    return dict(out=out.view(-1, n, d), dtable=grad[:v])


_EXACT = dict(xent=_exact_xent, q8_linear=_exact_q8_linear, q8_act=_exact_q8_act, norm=_exact_norm, embed=_exact_embed)
