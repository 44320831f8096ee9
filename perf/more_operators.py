"""Three operators of a transformer block's attention half, as a program built on
this library runs them through the C entry points of include/mle_hip.h.

A case is a dict of plain values; `kind` names the operator and the rest are its
sizes and options:

  attn    attention with a causal sliding window and a few first positions that
          stay visible (sinks), heads in groups that share keys and values,
          sequences padded to a common length: forward and backward
  step    the same for the newest tokens of each sequence over a cache of keys
          and values: one pass of sampling
  rotary  rotary positions with one to three axes on queries and keys: forward,
          and the gradient's inverse turn
  norm    layer norm with a weight and a bias after an optional residual Add:
          forward and backward

Tensors are float32, lengths and positions int32.  Gradients are assigned, as in
a step after zero_grad.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
EPS = 1e-5            # the norm's epsilon
NEIGHBOURS, BY_AXIS = 1, 2   # rotary flags
MAX_FLOPS = 2.0e11    # of a drawn case: the largest listed one's
MAX_BYTES = 2.1e9
MAX_SCORES = 5.4e8    # of a drawn case: heads x positions x positions of the plain form

# --------------------------------------------------------------------- cases


def listed() -> list[dict]:
    return [
        # Two short sentences of a small model: latency.
        dict(name="attn_small", kind="attn", batch=2, seq=64, heads=4, kv_heads=4, dim=32, window=64, sinks=0, padded=0),
        # The transformer block's attention, local: 32 x 256 tokens, 8 heads of 64.
        dict(name="attn_block", kind="attn", batch=32, seq=256, heads=8, kv_heads=8, dim=64, window=128, sinks=4, padded=0),
        # Padded sequences of no round size, heads of 80 in groups of three.
        dict(name="attn_ragged", kind="attn", batch=3, seq=777, heads=6, kv_heads=2, dim=80, window=200, sinks=3, padded=1),
        # Long documents, wide heads in groups of four.
        dict(name="attn_long", kind="attn", batch=2, seq=4096, heads=16, kv_heads=4, dim=128, window=1024, sinks=4, padded=0),
        # One conversation's next token: latency.
        dict(name="step_small", kind="step", batch=1, tokens=1, capacity=512, heads=8, kv_heads=8, dim=64, window=128, sinks=4),
        # A serving batch's next tokens over long caches.
        dict(name="step_batch", kind="step", batch=32, tokens=1, capacity=8192, heads=32, kv_heads=8, dim=128, window=4096,
             sinks=4),
        # The queries and keys of a sampling step.
        dict(name="rotary_step", kind="rotary", rows=32, heads=32, kv_heads=8, dim=128, sections="64", flags=0, far=100000),
        # The transformer block's queries and keys, image patches: rows and columns.
        dict(name="rotary_block", kind="rotary", rows=8192, heads=8, kv_heads=8, dim=64, sections="16,16", flags=BY_AXIS,
             far=256),
        # Video tokens: time, height and width share a head's pairs.
        dict(name="rotary_video", kind="rotary", rows=32768, heads=16, kv_heads=4, dim=128, sections="16,24,24", flags=0,
             far=1000000),
        # One short sequence: latency.
        dict(name="norm_small", kind="norm", rows=64, cols=256, residual=1),
        # The transformer block's residual stream.
        dict(name="norm_block", kind="norm", rows=8192, cols=512, residual=1),
        # A wide model's residual stream.
        dict(name="norm_wide", kind="norm", rows=16384, cols=4096, residual=1),
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng: random.Random) -> tuple[int, int]:
    kv = rng.choice((1, 2, 4, 8))
    return kv * rng.choice((1, 1, 2, 3, 4)), kv


def _dim(rng: random.Random) -> int:
    return rng.choice((16, 32, 40, 64, 64, 64, 72, 80, 96, 128, 128))


def _some_sections(rng: random.Random, dim: int) -> str:
    """Pairs of each axis; now and then a part of the head is left unturned."""
    pairs = dim // 2 if rng.random() < 0.75 else max(4, dim // 4)
    axes = rng.randint(1, 3)
    first = [max(1, pairs // axes + rng.randint(-1, 1)) for _ in range(axes - 1)]
    return ",".join(map(str, first + [pairs - sum(first)]))


def _sections(case: dict) -> list[int]:
    return [int(n) for n in case["sections"].split(",")]


def _draw_once(rng: random.Random) -> dict:
    kind = rng.choice(("attn", "attn", "attn", "attn", "step", "step", "rotary", "rotary", "norm", "norm"))
    if kind == "attn":
        heads, kv = _heads(rng)
        seq = _log_int(rng, 16, 4096)
        return dict(kind=kind, batch=_log_int(rng, 1, 32), seq=seq, heads=heads, kv_heads=kv, dim=_dim(rng),
                    window=_log_int(rng, 8, seq), sinks=rng.choice((0, 1, 4, rng.randint(2, 40))), padded=rng.randint(0, 1))
    if kind == "step":
        heads, kv = _heads(rng)
        cap = _log_int(rng, 64, 16384)
        return dict(kind=kind, batch=_log_int(rng, 1, 64), tokens=rng.choice((1, 1, 1, 2, 5)), capacity=cap, heads=heads,
                    kv_heads=kv, dim=_dim(rng), window=_log_int(rng, 16, cap), sinks=rng.choice((0, 4, rng.randint(1, 40))))
    if kind == "rotary":
        heads, kv = _heads(rng)
        dim = _dim(rng)
        return dict(kind=kind, rows=_log_int(rng, 1, 32768), heads=heads, kv_heads=kv, dim=dim, sections=_some_sections(rng, dim),
                    flags=rng.randint(0, 3), far=_log_int(rng, 64, 1000000))
    cols = _log_int(rng, 64, 8192)
    m = rng.choice((16, 16, 4, 1))
    return dict(kind=kind, rows=_log_int(rng, 16, 16384), cols=max(m, cols // m * m), residual=rng.randint(0, 1))


def draw(rng: random.Random) -> dict:
    while True:
        case = _draw_once(rng)
        w = work(case)
        scores = case["batch"] * case["heads"] * case["seq"] ** 2 if case["kind"] == "attn" else 0
        if w["flops"] <= MAX_FLOPS and w["bytes"] <= MAX_BYTES and scores <= MAX_SCORES:
            return case


def _seen(first: int, last: int, window: int, sinks: int) -> int:
    """Visible keys of the queries at positions first .. last - 1, together."""
    p = torch.arange(first, last, dtype=torch.int64)
    return int((torch.clamp(p + 1, max=window) + torch.clamp(p + 1 - window, min=0, max=sinks)).sum())


def work(case: dict) -> dict:
    c, k = case, case["kind"]
    if k == "attn":
        rows, d = c["batch"] * c["seq"], c["dim"]
        pairs = c["batch"] * c["heads"] * _seen(0, c["seq"], c["window"], c["sinks"])
        # q, out, dout, dq of every head, k, v, dk, dv of every group, lse
        return dict(flops=14.0 * d * pairs, bytes=4.0 * rows * (4 * c["heads"] * d + 4 * c["kv_heads"] * d + c["heads"]))
    if k == "step":
        t, d, cap = c["tokens"], c["dim"], c["capacity"]
        keys = min(cap, c["sinks"] + c["window"] + t - 1)
        pairs = c["batch"] * c["heads"] * _seen(cap - t, cap, c["window"], c["sinks"])
        return dict(flops=4.0 * d * pairs,
                    bytes=4.0 * c["batch"] * (2 * keys * c["kv_heads"] * d + 2 * t * c["heads"] * d))
    if k == "rotary":
        # both tensors read and written, forth and back; the positions twice
        n = c["rows"] * (c["heads"] + c["kv_heads"]) * c["dim"]
        return dict(flops=0.0, bytes=4.0 * (4 * n + 2 * c["rows"] * len(_sections(c))))
    n = c["rows"] * c["cols"]
    # x, the residual, h, dy and dres read; h, y and dh written
    return dict(flops=0.0, bytes=4.0 * (n * (5 + 3 * c["residual"]) + 4 * c["cols"] + 2 * c["rows"]))


# ------------------------------------------------------------------- prepare


def _normal(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV).mul_(scale)


def _new(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device=DEV)


def _ws(nbytes):
    return _new(max(int(nbytes), 16), dtype=torch.uint8)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = _PREPARE[case["kind"]](case, g)
    s["case"] = case
    return s


def _prep_attn(c, g):
    b, n, h, kv, d = c["batch"], c["seq"], c["heads"], c["kv_heads"], c["dim"]
    s = dict(q=_normal(g, b, n, h * d), k=_normal(g, b, n, kv * d), v=_normal(g, b, n, kv * d),
             dout=_normal(g, b, n, h * d, scale=1e-3), lengths=None)
    if c["padded"]:
        s["lengths"] = torch.randint(n // 3, n + 1, (b,), generator=g, device=DEV, dtype=torch.int32)
    if own:
        from ml_engine_amd import hip
        hip.init(0)
        s.update(out=_new(b, n, h * d), lse=_new(b, h, n), dq=_new(b, n, h * d), dk=_new(b, n, kv * d),
                 dv=_new(b, n, kv * d),
                 ws=_ws(hip.lib().mle_window_attention_ws_bytes(b, n, h, kv, d, c["window"], c["sinks"])))
    return s


def _prep_step(c, g):
    b, t, cap, h, kv, d = c["batch"], c["tokens"], c["capacity"], c["heads"], c["kv_heads"], c["dim"]
    # caches filled to different lengths, one of them wholly
    lengths = torch.randint(max(t, cap // 2), cap + 1, (b,), generator=g, device=DEV, dtype=torch.int32)
    lengths[0] = cap
    s = dict(q=_normal(g, b, t, h * d), k=_normal(g, b, cap, kv * d), v=_normal(g, b, cap, kv * d), lengths=lengths)
    if own:
        from ml_engine_amd import hip
        hip.init(0)
        s.update(out=_new(b, t, h * d),
                 ws=_ws(hip.lib().mle_window_attention_step_ws_bytes(b, t, cap, h, kv, d, c["window"], c["sinks"])))
    return s


def _prep_rotary(c, g):
    r, h, kv, d, a = c["rows"], c["heads"], c["kv_heads"], c["dim"], len(_sections(c))
    s = dict(q=_normal(g, r, h * d), k=_normal(g, r, kv * d), dq=_normal(g, r, h * d, scale=1e-3),
             dk=_normal(g, r, kv * d, scale=1e-3),
             positions=torch.randint(0, c["far"], (a, r), generator=g, device=DEV, dtype=torch.int32))
    if own:
        import ctypes

        from ml_engine_amd import hip
        hip.init(0)
        s.update(sections=(ctypes.c_int * a)(*_sections(c)), q1=_new(r, h * d), k1=_new(r, kv * d), dq1=_new(r, h * d),
                 dk1=_new(r, kv * d))
    return s


def _prep_norm(c, g):
    r, n = c["rows"], c["cols"]
    # rows of different size around a mean that is not zero
    s = dict(x=_normal(g, r, n) * (0.5 + torch.rand(r, 1, generator=g, device=DEV)) + 0.3,
             r=_normal(g, r, n) if c["residual"] else None, w=1.0 + _normal(g, n, scale=0.1), b=_normal(g, n, scale=0.1),
             dy=_normal(g, r, n, scale=1e-3), dres=_normal(g, r, n, scale=1e-3) if c["residual"] else None)
    if own:
        from ml_engine_amd import hip
        hip.init(0)
        s.update(h=_new(r, n), y=_new(r, n), mean=_new(r), rstd=_new(r), dh=_new(r, n), dw=_new(n), db=_new(n),
                 ws=_ws(hip.lib().mle_add_layernorm_ws_bytes(r, n)))
    return s


_PREPARE = dict(attn=_prep_attn, step=_prep_step, rotary=_prep_rotary, norm=_prep_norm)

# ----------------------------------------------------------------------- run


def run(state: dict):
    k = state["case"]["kind"]
    return _OWN[k](state, state["case"]) if own else _PLAIN[k](state, state["case"])


def _p(t):
    return None if t is None else t.data_ptr()


def _scale(c):
    return 1.0 / math.sqrt(c["dim"])


def _own_attn(s, c):
    from ml_engine_amd import hip
    b, n, h, kv, d = c["batch"], c["seq"], c["heads"], c["kv_heads"], c["dim"]
    e, f = h * d, kv * d
    hip.call("mle_window_attention_fwd", None, _p(s["q"]), e, _p(s["k"]), f, _p(s["v"]), f, _p(s["out"]), e, _p(s["lse"]),
             _p(s["lengths"]), b, n, h, kv, d, _scale(c), c["window"], c["sinks"])
    hip.call("mle_window_attention_bwd", None, _p(s["q"]), e, _p(s["k"]), f, _p(s["v"]), f, _p(s["out"]), e, _p(s["lse"]),
             _p(s["dout"]), e, _p(s["dq"]), e, 0, _p(s["dk"]), f, 0, _p(s["dv"]), f, 0, _p(s["lengths"]), b, n, h, kv, d,
             _scale(c), c["window"], c["sinks"], _p(s["ws"]), s["ws"].numel())
    return {k: s[k] for k in ("out", "lse", "dq", "dk", "dv")}


def _own_step(s, c):
    from ml_engine_amd import hip
    b, t, cap, h, kv, d = c["batch"], c["tokens"], c["capacity"], c["heads"], c["kv_heads"], c["dim"]
    hip.call("mle_window_attention_step", None, _p(s["q"]), h * d, _p(s["k"]), kv * d, _p(s["v"]), kv * d, _p(s["out"]),
             h * d, _p(s["lengths"]), b, t, cap, h, kv, d, _scale(c), c["window"], c["sinks"], _p(s["ws"]), s["ws"].numel())
    return s["out"]


def _own_rotary(s, c):
    from ml_engine_amd import hip
    r, h, kv, d, a = c["rows"], c["heads"], c["kv_heads"], c["dim"], len(_sections(c))
    for inverse, q, k, q1, k1 in ((0, "q", "k", "q1", "k1"), (1, "dq", "dk", "dq1", "dk1")):
        hip.call("mle_rotary", None, r, d, _p(s[q]), h * d, _p(s[q1]), h * d, h, _p(s[k]), kv * d, _p(s[k1]), kv * d, kv,
                 _p(s["positions"]), a, s["sections"], 10000.0, c["flags"], inverse, 0)
    return {k: s[k] for k in ("q1", "k1", "dq1", "dk1")}


def _own_norm(s, c):
    from ml_engine_amd import hip
    r, n = c["rows"], c["cols"]
    h = s["h"] if c["residual"] else s["x"]  # without a residual x is what the backward reads
    hip.call("mle_add_layernorm_fwd", None, r, n, _p(s["x"]), _p(s["r"]), _p(s["w"]), _p(s["b"]), EPS,
             _p(h) if c["residual"] else None, _p(s["y"]), _p(s["mean"]), _p(s["rstd"]))
    hip.call("mle_add_layernorm_bwd", None, r, n, _p(h), _p(s["w"]), _p(s["mean"]), _p(s["rstd"]), _p(s["dy"]),
             _p(s["dres"]), _p(s["dh"]), 0, _p(s["dw"]), _p(s["db"]), 0, _p(s["ws"]), s["ws"].numel())
    return dict(h=h, y=s["y"], mean=s["mean"], rstd=s["rstd"], dh=s["dh"], dw=s["dw"], db=s["db"])


_OWN = dict(attn=_own_attn, step=_own_step, rotary=_own_rotary, norm=_own_norm)

# ---------------------------------------------------------------- plain form


def _split(x, heads, repeat):
    """[batch, rows, heads * dim] as [batch, heads * repeat, rows, dim], each head `repeat` times."""
    b, n, e = x.shape
    return x.view(b, n, heads, e // heads).transpose(1, 2).repeat_interleave(repeat, 1)


def _join(x, heads):
    """The other way, the gradients of a shared head added."""
    b, h, n, d = x.shape
    return x.view(b, heads, h // heads, n, d).sum(2).transpose(1, 2).reshape(b, n, heads * d)


def _hidden(pos, keys, lengths, window, sinks):
    """Keys that take no part for the query at pos [..., rows, 1], keys [columns]."""
    return (keys > pos) | ((pos - keys >= window) & (keys >= sinks)) | (keys >= lengths)


def _plain_attn(s, c):
    b, n, h, kv = c["batch"], c["seq"], c["heads"], c["kv_heads"]
    q, dout = _split(s["q"], h, 1), _split(s["dout"], h, 1)
    k, v = _split(s["k"], kv, h // kv), _split(s["v"], kv, h // kv)
    at = torch.arange(n, device=DEV)
    lengths = at.new_full((b,), n) if s["lengths"] is None else s["lengths"].long()
    lengths = lengths.view(b, 1, 1, 1)
    live = at[:, None] < lengths                     # queries that are there
    hidden = _hidden(at[:, None], at, lengths, c["window"], c["sinks"]) | ~live
    x = (q @ k.transpose(2, 3)).mul_(_scale(c)).masked_fill_(hidden, -math.inf)
    top = x.amax(3, keepdim=True).clamp_(min=-3e38)  # of a row without keys: finite
    p = x.sub_(top).exp_()
    total = p.sum(3, keepdim=True)
    lse = (top + total.log()).masked_fill(~live, -math.inf).squeeze(3)
    p.div_(total.masked_fill(~live, 1.0))
    out = p @ v
    dv = p.transpose(2, 3) @ dout
    ds = dout @ v.transpose(2, 3)
    ds.sub_((dout * out).sum(3, keepdim=True)).mul_(p).mul_(_scale(c))
    dq, dk = ds @ k, ds.transpose(2, 3) @ q
    return dict(out=_join(out, h), lse=lse, dq=_join(dq, h), dk=_join(dk, kv), dv=_join(dv, kv))


def _plain_step(s, c):
    b, t, cap, h, kv = c["batch"], c["tokens"], c["capacity"], c["heads"], c["kv_heads"]
    q = _split(s["q"], h, 1)
    k, v = _split(s["k"], kv, h // kv), _split(s["v"], kv, h // kv)
    lengths = s["lengths"].long().view(b, 1, 1, 1)
    pos = lengths - t + torch.arange(t, device=DEV)[:, None]
    hidden = _hidden(pos, torch.arange(cap, device=DEV), lengths, c["window"], c["sinks"])
    x = (q @ k.transpose(2, 3)).mul_(_scale(c)).masked_fill_(hidden, -math.inf)
    p = x.sub_(x.amax(3, keepdim=True)).exp_()
    return _join(p.div_(p.sum(3, keepdim=True)) @ v, h)


def _frequencies(c):
    """Axis and frequency of each pair of a head."""
    sec = _sections(c)
    axis = torch.repeat_interleave(torch.arange(len(sec)), torch.tensor(sec))
    if c["flags"] & BY_AXIS:
        start = torch.cumsum(torch.tensor([0] + sec[:-1]), 0)
        i, n = torch.arange(sum(sec)) - start[axis], torch.tensor(sec)[axis]
    else:
        i, n = torch.arange(sum(sec)), torch.full((sum(sec),), sum(sec))
    return axis.to(DEV), torch.pow(10000.0, -i.double() / n.double()).to(DEV)


def _pairs(c):
    """Places of the first and the second value of each pair in a head."""
    i = torch.arange(sum(_sections(c)), device=DEV)
    return (2 * i, 2 * i + 1) if c["flags"] & NEIGHBOURS else (i, i + sum(_sections(c)))


def _turn(x, heads, cos, sin, places):
    v = x.view(x.shape[0], heads, -1)
    a, b = v[:, :, places[0]], v[:, :, places[1]]
    y = v.clone()
    y[:, :, places[0]] = a * cos - b * sin
    y[:, :, places[1]] = a * sin + b * cos
    return y.view_as(x)


def _plain_rotary(s, c):
    h, kv = c["heads"], c["kv_heads"]
    axis, freq = _frequencies(c)
    angle = s["positions"].double()[axis].t() * freq  # 64 bits: far positions
    cos, sin, at = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :], _pairs(c)
    return dict(q1=_turn(s["q"], h, cos, sin, at), k1=_turn(s["k"], kv, cos, sin, at), dq1=_turn(s["dq"], h, cos, -sin, at),
                dk1=_turn(s["dk"], kv, cos, -sin, at))


def _plain_norm(s, c):
    h = s["x"] + s["r"] if c["residual"] else s["x"]
    mean = h.mean(1, keepdim=True)
    u = h - mean
    rstd = 1.0 / (u.square().mean(1, keepdim=True) + EPS).sqrt()
    u = u * rstd
    y = u * s["w"] + s["b"]
    g = s["dy"] * s["w"]
    dh = rstd * (g - g.mean(1, keepdim=True) - u * (g * u).mean(1, keepdim=True))
    if s["dres"] is not None:
        dh = dh + s["dres"]
    return dict(h=h, y=y, mean=mean.squeeze(1), rstd=rstd.squeeze(1), dh=dh, dw=(s["dy"] * u).sum(0), db=s["dy"].sum(0))


_PLAIN = dict(attn=_plain_attn, step=_plain_step, rotary=_plain_rotary, norm=_plain_norm)

# --------------------------------------------------------------------- exact


def exact(case: dict, seed: int):
    """What run() returns for prepare(case, seed), in 64 bits."""
    s = prepare(case, seed)
    return _EXACT[case["kind"]](s, case)


def _exact_one(q, k, v, first, c):
    """Outputs and log-sums of queries [heads, rows, dim] at positions first, first + 1, ... against
    keys and values [keys, dim]; autograd goes through it."""
    i = torch.arange(q.shape[1], device=DEV)[:, None] + first
    j = torch.arange(k.shape[0], device=DEV)[None, :]
    seen = torch.logical_and(j <= i, torch.logical_or(i - j < c["window"], j < c["sinks"]))
    x = torch.where(seen, torch.matmul(q, k.t()) / math.sqrt(c["dim"]), torch.full((), -math.inf, device=DEV).double())
    lse = torch.logsumexp(x, 2)
    return torch.matmul(torch.exp(x - lse[:, :, None]), v), lse


def _exact_attn(s, c):
    b, n, h, kv, d = c["batch"], c["seq"], c["heads"], c["kv_heads"], c["dim"]
    g = h // kv
    out, dq = (torch.zeros(b, n, h, d, dtype=torch.float64, device=DEV) for _ in range(2))
    dk, dv = (torch.zeros(b, n, kv, d, dtype=torch.float64, device=DEV) for _ in range(2))
    lse = torch.full((b, h, n), -math.inf, dtype=torch.float64, device=DEV)
    ends = [n] * b if s["lengths"] is None else s["lengths"].tolist()
    for i, m in enumerate(ends):
        for e in range(kv):
            heads = slice(e * g, (e + 1) * g)
            q = s["q"].view(b, n, h, d)[i, :m, heads].transpose(0, 1).double().requires_grad_(True)
            k = s["k"].view(b, n, kv, d)[i, :m, e].double().requires_grad_(True)
            v = s["v"].view(b, n, kv, d)[i, :m, e].double().requires_grad_(True)
            y, ls = _exact_one(q, k, v, 0, c)
            up = s["dout"].view(b, n, h, d)[i, :m, heads].transpose(0, 1).double()
            gq, gk, gv = torch.autograd.grad(y, (q, k, v), up)
            out[i, :m, heads], dq[i, :m, heads] = y.detach().transpose(0, 1), gq.transpose(0, 1)
            dk[i, :m, e], dv[i, :m, e], lse[i, heads, :m] = gk, gv, ls.detach()
    return dict(out=out.view(b, n, h * d), lse=lse, dq=dq.view(b, n, h * d), dk=dk.view(b, n, kv * d),
                dv=dv.view(b, n, kv * d))


def _exact_step(s, c):
    b, t, cap, h, kv, d = c["batch"], c["tokens"], c["capacity"], c["heads"], c["kv_heads"], c["dim"]
    g = h // kv
    out = torch.zeros(b, t, h, d, dtype=torch.float64, device=DEV)
    for i, m in enumerate(s["lengths"].tolist()):
        for e in range(kv):
            heads = slice(e * g, (e + 1) * g)
            q = s["q"].view(b, t, h, d)[i, :, heads].transpose(0, 1).double()
            k, v = (s[x].view(b, cap, kv, d)[i, :m, e].double() for x in "kv")
            out[i, :, heads] = _exact_one(q, k, v, m - t, c)[0].transpose(0, 1)
    return out.view(b, t, h * d)


def _exact_rotary(s, c):
    sec, pairs = _sections(c), sum(_sections(c))
    angles = []
    for a, n in enumerate(sec):
        i = torch.arange(n, device=DEV, dtype=torch.float64)
        e = i / n if c["flags"] & BY_AXIS else (i + sum(sec[:a])) / pairs
        angles.append(s["positions"][a].double()[:, None] * torch.exp(-math.log(10000.0) * e)[None, :])
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), torch.cat(angles, 1))[:, None, :]

    def go(x, heads, by):
        v = x.double().view(x.shape[0], heads, -1)
        r, rest = v[:, :, :2 * pairs], v[:, :, 2 * pairs:]
        if c["flags"] & NEIGHBOURS:
            z = torch.view_as_complex(r.reshape(*r.shape[:2], pairs, 2).contiguous()) * by
            r = torch.view_as_real(z).reshape(r.shape)
        else:
            z = torch.complex(r[:, :, :pairs].contiguous(), r[:, :, pairs:].contiguous()) * by
            r = torch.cat([z.real, z.imag], 2)
        return torch.cat([r, rest], 2).view(x.shape)

    h, kv = c["heads"], c["kv_heads"]
    return dict(q1=go(s["q"], h, turn), k1=go(s["k"], kv, turn), dq1=go(s["dq"], h, turn.conj()),
                dk1=go(s["dk"], kv, turn.conj()))


def _exact_norm(s, c):
    # the sum is held in 32 bits: what is normed, and what the backward reads
    h = (s["x"].double() + s["r"].double()).float().double() if c["residual"] else s["x"].double()
    h.requires_grad_(True)
    w, b = s["w"].double().requires_grad_(True), s["b"].double().requires_grad_(True)
    var, mean = torch.var_mean(h, 1, unbiased=False, keepdim=True)
    rstd = torch.rsqrt(var + EPS)
    y = (h - mean) * rstd * w + b
    dh, dw, db = torch.autograd.grad(y, (h, w, b), s["dy"].double())
    if s["dres"] is not None:
        dh = dh + s["dres"].double()
    return dict(h=h.detach(), y=y.detach(), mean=mean.detach().squeeze(1), rstd=rstd.detach().squeeze(1), dh=dh, dw=dw, db=db)


_EXACT = dict(attn=_exact_attn, step=_exact_step, rotary=_exact_rotary, norm=_exact_norm)
