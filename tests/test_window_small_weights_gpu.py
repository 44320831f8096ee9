"""Windowed attention where a row's or a key's largest probability (and dS) meets zeros, so that its
results are made of the smallest: each is held to the bits of its own size, not of the largest's."""
import numpy as np
import pytest

from conftest import rng
from test_window_attention_gpu import Case

pytestmark = pytest.mark.gpu
U = 2.0 ** -24        # half a step of fp32
PRODUCT = 2.0 ** -21  # of a product of two operands in two fp16 parts: 2^-23 each, 2^-22 without lo lo
WEIGHT = 2.0 ** -23   # of P or dS as an operand, or, if that is more,
FLOOR = 2.0 ** -36    # of the largest in its row (column): 2^-25 where that is at 2^12 or above, and rows' unlike powers of two
ROW = 40


def build(hip, dim, heads=1, n=700):
    """Row ROW's weights lie on keys 0 and 1, half each; all other keys have 2^-24 of them.  Those two keys
    have a weight of some 2^-24 of that in all other rows.  What the large weights multiply is zero from column 1 on."""
    def spoil(c):
        r = rng(dim)
        some = lambda a: (1 + 0.3 * r.standard_normal(a.shape)).astype(np.float32)  # noqa: E731
        c.q[:], c.k[:], c.v[:], c.dout[:] = 0.5 * some(c.q), 0.5 * some(c.k), some(c.v), some(c.dout)
        level = c.scale * 0.25 * (dim - 1)  # the other scores, about
        c.k[..., 0] = 0
        c.k[:, :2], c.v[:, :2] = 0, 0
        c.k[:, :2, :, 0] = 4
        c.v[:, 0, :, 0], c.v[:, 1, :, 0] = 1, -1
        c.q[..., 0] = (level - 13) / (4 * c.scale)
        c.q[:, ROW] = 0
        c.q[:, ROW, :, 0] = 16.6 / (4 * c.scale)
        c.dout[..., 0] *= 0.3
        c.dout[:, ROW, :, 1:] = 0
        c.dout[:, :2] = 0  # (rows that see nothing else)
    c = Case(hip, 1, n, heads, 1, dim, n, 0, spoil=spoil)
    return c


def bounds(c):
    """Results in 64 bits and how far from them operands and sums of these bits may be, from column 1 on."""
    b, n, heads, _, dim = c.dims
    f = lambda a: a.astype(np.float64)  # noqa: E731
    k, v, s = f(c.k[0, :, 0]), f(c.v[0, :, 0]), abs(c.scale)
    see = np.tril(np.ones((n, n), bool))
    r = {"out": [], "dq": [], "dk": 0, "dv": 0, "e_out": [], "e_dq": [], "e_dk": 0, "e_dv": 0}
    count = see.sum(1, keepdims=True)
    rows = see.sum(0)[:, None]
    for h in range(heads):
        q, g = f(c.q[0, :, h]), f(c.dout[0, :, h])
        x = np.where(see, c.scale * (q @ k.T), -np.inf)
        m = x.max(1, keepdims=True)
        lse = m + np.log(np.exp(x - m).sum(1, keepdims=True))
        p = np.exp(x - lse)
        # a score: its products and sums; below 2^-39 of a tile's largest nothing of K and Q
        big = lambda a, c: np.abs(a).max(1, keepdims=True) * np.abs(c).max()  # noqa: E731
        dot = lambda a, c: (PRODUCT + (dim + 8) * U) * (np.abs(a) @ np.abs(c).T) + 2.0 ** -38 * dim * big(a, c)  # noqa: E731
        # .. its place in the exponent and that of lse, exp2 to two steps
        ex = s * dot(q, k) + 4 * U * (np.abs(np.where(see, x, 0)) + np.abs(lse)) + 4 * U
        el = (p * ex).sum(1, keepdims=True) + (count + 16) * U
        ep = (ex + el) * p
        out = p @ v
        wide = p.max(1, keepdims=True)
        sums = (count + 16) * U + 2.0 ** -22 + WEIGHT
        eout = ep @ np.abs(v) + sums * (p @ np.abs(v)) + (FLOOR * wide * see) @ np.abs(v) + 2.0 ** -38 * np.abs(v).max() * p.sum(1, keepdims=True)
        dp = g @ v.T
        delta = (g * out).sum(1, keepdims=True)
        edelta = (np.abs(g) * eout).sum(1, keepdims=True) + (dim + 8) * U * (np.abs(g) * np.abs(out)).sum(1, keepdims=True)
        ds = p * (dp - delta)
        eds = ep * np.abs(dp - delta) + p * (dot(g, v) + edelta + 4 * U * (np.abs(dp) + np.abs(delta)))
        ads = np.abs(ds)
        edq = s * (eds @ np.abs(k) + sums * (ads @ np.abs(k)) + (FLOOR * ads.max(1, keepdims=True) * see) @ np.abs(k) + 2.0 ** -38 * np.abs(k).max() * ads.sum(1, keepdims=True))
        # a row's dout is at a power of two of its own, which its P takes up
        size = np.abs(g).max(1, keepdims=True)
        sums = (rows + 16) * U + 2.0 ** -22 + WEIGHT
        edk = s * (eds.T @ np.abs(q) + sums * (ads.T @ np.abs(q)) + FLOOR * ads.max(0)[:, None] * (see.T @ np.abs(q)) + 2.0 ** -38 * np.abs(q).max() * ads.sum(0)[:, None])
        edv = ep.T @ np.abs(g) + sums * (p.T @ np.abs(g)) + FLOOR * (p * size).max(0)[:, None] * rows + 2.0 ** -38 * (p * size).sum(0)[:, None]
        r["out"].append(out), r["e_out"].append(eout), r["dq"].append(c.scale * (ds @ k)), r["e_dq"].append(edq)
        r["dk"] = r["dk"] + c.scale * (ds.T @ q)
        r["dv"] = r["dv"] + p.T @ g
        r["e_dk"], r["e_dv"] = r["e_dk"] + edk, r["e_dv"] + edv
    for key in ("out", "e_out", "dq", "e_dq"):
        r[key] = np.stack(r[key], 1)
    for key in ("dk", "dv", "e_dk", "e_dv"):
        r[key] = r[key][:, None]
    return r


@pytest.mark.parametrize("dim,heads", [(64, 1), (40, 2), (80, 1), (128, 2)])
def test_results_of_the_smallest_weights(hip, dim, heads):
    c = build(hip, dim, heads)
    c.forward()
    c.backward()
    got, r = c.results(), bounds(c)
    for name, at in (("out", slice(ROW, ROW + 1)), ("dq", slice(ROW, ROW + 1)), ("dk", slice(0, 2)), ("dv", slice(0, 2))):
        err = np.abs(got[name][0, at, :, 1:] - r[name][at, :, 1:])
        assert (err <= r["e_" + name][at, :, 1:]).all(), (name, float((err / r["e_" + name][at, :, 1:]).max()))


@pytest.mark.parametrize("dim,seq", [(64, 600), (128, 300), (80, 40), (64, 3000)])
def test_log_sum_of_even_rows(hip, dim, seq):
    """Queries of zeros: every sum is a whole number of equal weights, exact, so that lse is log(count) but for
    its own rounding, 2^-24 of it, and that of the logarithm of a number's fraction, one step of 2^-23."""
    def spoil(c):
        c.q[:] = 0
    c = Case(hip, 1, seq, 1, 1, dim, seq, 0, spoil=spoil)
    c.forward()
    want = np.log(np.arange(1, seq + 1))
    assert (np.abs(c.lse.numpy()[0, 0] - want) <= U * want + 2 * U).all()
