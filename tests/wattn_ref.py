"""Windowed attention with sinks in 64 bits, and how far kernels that hold their
products' operands in 22 bits and their sums in fp32 may be from it."""
import math

import numpy as np

F32 = 2.0 ** -24   # half a step of fp32
OP = 2.0 ** -22    # an operand in 22 bits, rounded or truncated
FLOOR = 2.0 ** -36  # of a tile's largest product: operands far below the largest


def visible(pos, n, window, sinks):
    j = np.arange(n)[None, :]
    p = pos[:, None]
    return (j <= p) & ((p - j < window) | (j < sinks))


def _dot_error(a, b):
    """Bound of the error of a b^T (a [m, d], b [n, d]): operands, sums, and what lies far below the largest."""
    d = a.shape[1]
    size = np.abs(a) @ np.abs(b).T
    return (2 * OP + (d + 8) * F32) * size + FLOOR * d * (np.abs(a).max(initial=0) * np.abs(b).max(initial=0))


def head(q, k, v, pos, window, sinks, scale, dout=None):
    """One head of one sequence: rows of q at positions pos over keys [n].  Returns values and bounds."""
    n = k.shape[0]
    see = visible(pos, n, window, sinks)
    k, v = (np.where(see.any(0)[:, None], a, 0) for a in (k, v))  # what no row sees, whatever it holds
    x = np.where(see, scale * (q @ k.T), -np.inf)
    m = x.max(1, keepdims=True)
    e = np.exp(x - m)
    lse = m + np.log(e.sum(1, keepdims=True))
    p = np.exp(x - lse)
    out = p @ v
    ex = np.where(see, abs(scale) * _dot_error(q, k), 0) + 4 * F32 * np.where(see, np.abs(x) + np.abs(lse), 0)
    count = see.sum(1, keepdims=True)
    elog = ex.max(1, keepdims=True) + (count + 16) * F32
    ep = 2 * (ex + elog + 8 * F32) * p  # (2: second order)
    big = np.where(see[:, :, None], np.abs(v)[None], 0).max(1)  # largest value that a row sees
    eout = ep @ np.abs(v) + (2 * OP + (count + 16) * F32) * (p @ np.abs(v)) + FLOOR * big
    r = dict(out=out, lse=lse[:, 0], e_out=eout, e_lse=elog[:, 0] + 2 * F32 * np.abs(lse[:, 0]))
    if dout is None:
        return r
    dp = np.where(see, dout @ v.T, 0)
    delta = (dout * out).sum(1, keepdims=True)
    edelta = (np.abs(dout) * eout).sum(1, keepdims=True) + (q.shape[1] + 8) * F32 * (np.abs(dout) * np.abs(out)).sum(1, keepdims=True)
    ds = p * (dp - delta)
    edp = np.where(see, _dot_error(dout, v), 0)
    eds = p * (edp + edelta) + ep * np.abs(dp - delta) + 8 * F32 * p * (np.abs(dp) + np.abs(delta))
    rows = see.sum(0)[:, None]  # of each key
    r["dq"] = scale * (ds @ k)
    r["dk"] = scale * (ds.T @ q)
    r["dv"] = p.T @ dout
    s = abs(scale)
    r["e_dq"] = s * (eds @ np.abs(k) + (2 * OP + (count + 16) * F32) * (np.abs(ds) @ np.abs(k)) + FLOOR * (p * (np.abs(dp) + np.abs(delta))).max(1, keepdims=True) * np.abs(k).max())
    r["e_dk"] = s * (eds.T @ np.abs(q) + (2 * OP + (rows + 16) * F32) * (np.abs(ds).T @ np.abs(q)) + FLOOR * np.abs(q).max() * (p * (np.abs(dp) + np.abs(delta))).max(0)[:, None])
    r["e_dv"] = ep.T @ np.abs(dout) + (2 * OP + (rows + 16) * F32) * (p.T @ np.abs(dout)) + FLOOR * np.abs(dout).max() * p.max(0)[:, None]
    return r


def whole(q, k, v, lengths, heads, kv_heads, window, sinks, scale, dout=None, at_end=False):
    """[batch, rows, heads, dim] and [batch, keys, kv_heads, dim], fp32 arrays; entries past a length are not read."""
    B, n, H, D = q.shape
    m = k.shape[1]
    g = heads // kv_heads
    r = {}
    z = lambda *s: np.zeros(s)  # noqa: E731
    for key in ("out", "e_out", "dq", "e_dq"):
        r[key] = z(B, n, H, D)
    for key in ("dk", "dv", "e_dk", "e_dv"):
        r[key] = z(B, m, kv_heads, D)
    r["lse"], r["e_lse"] = np.full((B, H, n), -np.inf), z(B, H, n)
    f = lambda a: a.astype(np.float64)  # noqa: E731
    for b in range(B):
        L = m if lengths is None else int(min(max(lengths[b], 0), m))
        pos = np.arange(n) + (L - n if at_end else 0)
        live = np.nonzero((pos >= 0) & (pos < L))[0]
        if len(live) == 0:
            continue
        for h in range(heads):
            e = h // g
            t = head(f(q[b, live, h]), f(k[b, :L, e]), f(v[b, :L, e]), pos[live], window, sinks, scale,
                     None if dout is None else f(dout[b, live, h]))
            r["out"][b, live, h], r["e_out"][b, live, h] = t["out"], t["e_out"]
            r["lse"][b, h, live], r["e_lse"][b, h, live] = t["lse"], t["e_lse"]
            if dout is not None:
                r["dq"][b, live, h], r["e_dq"][b, live, h] = t["dq"], t["e_dq"]
                for key in ("dk", "dv", "e_dk", "e_dv"):
                    r[key][b, :L, e] += t[key]
    return r


def check(got, r, name, old=None):
    """got against r[name] (added to old), within r's bound and the sum's own rounding."""
    want = r[name] + (0 if old is None else old.astype(np.float64))
    tol = r["e_" + name] + (0 if old is None else 2 * F32 * (np.abs(old) + np.abs(r[name])))
    assert got.shape == want.shape
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]), name
    err = np.abs(got[~inf] - want[~inf])
    bad = ~(err <= tol[~inf] + 1e-42)
    assert not bad.any(), (name, int(bad.sum()), float(np.nanmax(err / (tol[~inf] + 1e-42))), np.argwhere(~inf)[np.argmax(bad.ravel())])


def scale_of(dim):
    return float(np.float32(1.0 / math.sqrt(dim)))
