"""The residual Add with the layer norm, its weight and its bias, against 64 bits."""
import numpy as np
import pytest

from conftest import rng

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -24  # half a step of fp32
EPS = 1e-5


def at(hip, a, shift):
    """A device copy of a that begins `shift` floats into its buffer."""
    b = hip.Buffer.from_array(np.concatenate([np.zeros(shift, np.float32), a.reshape(-1).astype(np.float32)]))
    return b, b.ptr + 4 * shift


def norm64(h):
    h = h.astype(np.float64)
    mean = h.mean(1, keepdims=True)
    rstd = 1 / np.sqrt(((h - mean) ** 2).mean(1, keepdims=True) + np.float64(np.float32(EPS)))
    return mean, rstd, (h - mean) * rstd


SHAPES = [(1, 1), (1, 32), (3, 31), (5, 33), (64, 256), (7, 330), (130, 512), (9, 1000), (33, 1024), (6, 1500), (40, 2048),
          (3, 2052), (5, 4096), (2, 6001), (3, 8192), (2, 8200), (3, 20001), (1500, 64), (4, 7), (6, 37), (5, 2049), (2, 8191),
          (2500, 3), (255, 100), (256, 2048), (257, 40)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("residual,weight,acc,shift", [(1, 1, 0, 0), (0, 1, 1, 0), (1, 0, 1, 1)])
def test_forward_and_backward(hip, rows, cols, residual, weight, acc, shift):
    r = rng(rows * 31 + cols)
    x, res, dy, dres = (r.standard_normal((rows, cols)).astype(np.float32) for _ in range(4))
    x += r.uniform(-2, 2, (rows, 1)).astype(np.float32)
    w, b = (1 + 0.2 * r.standard_normal(cols)).astype(np.float32), r.standard_normal(cols).astype(np.float32)
    old_dh = r.standard_normal((rows, cols)).astype(np.float32)
    old_dw, old_db = (r.standard_normal(cols).astype(np.float32) for _ in range(2))
    bx, px = at(hip, x, shift)
    br, pr = at(hip, res, shift)
    bw, pw = at(hip, w, shift)
    bb, pb = at(hip, b, shift)
    bh, ph = at(hip, np.zeros((rows, cols)), shift)
    by, py = at(hip, np.zeros((rows, cols)), shift)
    gm, gs = hip.Buffer.empty(rows), hip.Buffer.empty(rows)
    hip.call("mle_add_layernorm_fwd", None, rows, cols, px, pr if residual else None, pw if weight else None,
             pb if weight else None, EPS, ph, py, gm.ptr, gs.ptr)
    h = bh.numpy().reshape(-1)[shift:].reshape(rows, cols)
    y = by.numpy().reshape(-1)[shift:].reshape(rows, cols)
    assert np.array_equal(h, x + res if residual else x)
    mean, rstd, u = norm64(h)
    w64, b64 = (w.astype(np.float64), b.astype(np.float64)) if weight else (np.ones(cols), np.zeros(cols))
    # statistics in 64 bits (centred values round once before they are squared)
    spread = np.abs(h.astype(np.float64)).max(1)
    assert (np.abs(gm.numpy() - mean[:, 0]) <= 2 * F32 * np.abs(mean[:, 0]) + 1e-12 * spread).all()
    assert (np.abs(gs.numpy() - rstd[:, 0]) <= 4 * F32 * rstd[:, 0]).all()
    # u rounds, then the product with the sum; rstd's own share
    assert (np.abs(y - (u * w64 + b64)) <= 4 * F32 * (np.abs(u * w64) + np.abs(b64)) + 1e-11 * spread[:, None] * rstd * np.abs(w64)).all()

    bdy, pdy = at(hip, dy, shift)
    bdr, pdr = at(hip, dres, shift)
    bdh, pdh = at(hip, old_dh, shift)
    gdw, gdb = hip.Buffer.from_array(old_dw), hip.Buffer.from_array(old_db)
    ws = hip.Buffer(hip.lib().mle_add_layernorm_ws_bytes(rows, cols))
    hip.call("mle_add_layernorm_bwd", None, rows, cols, ph, pw if weight else None, gm.ptr, gs.ptr, pdy,
             pdr if residual else None, pdh, acc, gdw.ptr, gdb.ptr, acc, ws.ptr, ws.nbytes)
    g = dy.astype(np.float64) * w64
    m1, m2 = g.mean(1, keepdims=True), (g * u).mean(1, keepdims=True)
    dh = rstd * (g - m1 - u * m2) + (dres if residual else 0) + (old_dh if acc else 0)
    got = bdh.numpy().reshape(-1)[shift:].reshape(rows, cols)
    # u from the rounded mean and rstd: half a step of the mean and of h's size, three of u's
    eu = F32 * (rstd * (np.abs(mean) + np.abs(h)) + 4 * np.abs(u))
    size = rstd * (np.abs(g) + np.abs(g).mean(1, keepdims=True) + np.abs(u) * np.abs(g * u).mean(1, keepdims=True))
    spill = rstd * (eu * np.abs(g * u).mean(1, keepdims=True) + np.abs(u) * (np.abs(g) * eu).mean(1, keepdims=True))
    assert (np.abs(got - dh) <= 12 * F32 * (size + np.abs(dres) + np.abs(old_dh)) + 2 * spill).all()
    dw = (dy * u).sum(0) + (old_dw if acc else 0)
    db = dy.astype(np.float64).sum(0) + (old_db if acc else 0)
    assert (np.abs(gdw.numpy() - dw) <= F32 * ((rows + 8) * np.abs(dy * u).sum(0) + 2 * np.abs(old_dw)) + (np.abs(dy) * eu).sum(0)).all()
    assert (np.abs(gdb.numpy() - db) <= F32 * ((rows + 8) * np.abs(dy).sum(0) + 2 * np.abs(old_db))).all()


def test_mean_far_above_the_spread(hip):
    """Rows of values near 1000 that differ by some 0.01: y keeps what their differences hold."""
    x = (1000 + 0.01 * rng(8).standard_normal((40, 700))).astype(np.float32)
    gx, gy, gm, gs = hip.Buffer.from_array(x), hip.Buffer.empty((40, 700)), hip.Buffer.empty(40), hip.Buffer.empty(40)
    hip.call("mle_add_layernorm_fwd", None, 40, 700, gx.ptr, None, None, None, EPS, None, gy.ptr, gm.ptr, gs.ptr)
    _, rstd, u = norm64(x)
    assert (np.abs(gy.numpy() - u) <= 6 * F32 * np.abs(u) + 1e-6 * F32).all()
    assert (np.abs(gs.numpy() - rstd[:, 0]) <= 4 * F32 * rstd[:, 0]).all()


def test_optional_outputs(hip):
    """h, y, dw and db can each be left out; what stays is the same."""
    r = rng(2)
    n = (40, 200)
    x, res, dy = (r.standard_normal(n).astype(np.float32) for _ in range(3))
    w, b = (r.standard_normal(200).astype(np.float32) for _ in range(2))
    gx, gr, gdy, gw, gb = (hip.Buffer.from_array(a) for a in (x, res, dy, w, b))
    h, y, m, s, y1, h1 = (hip.Buffer.empty(k) for k in (n, n, 40, 40, n, n))
    hip.call("mle_add_layernorm_fwd", None, 40, 200, gx.ptr, gr.ptr, gw.ptr, gb.ptr, EPS, h.ptr, y.ptr, m.ptr, s.ptr)
    hip.call("mle_add_layernorm_fwd", None, 40, 200, gx.ptr, gr.ptr, gw.ptr, gb.ptr, EPS, None, y1.ptr, m.ptr, s.ptr)
    hip.call("mle_add_layernorm_fwd", None, 40, 200, gx.ptr, gr.ptr, gw.ptr, gb.ptr, EPS, h1.ptr, None, m.ptr, s.ptr)
    assert np.array_equal(y.numpy(), y1.numpy()) and np.array_equal(h.numpy(), h1.numpy())
    hip.call("mle_add_layernorm_fwd", None, 40, 200, gx.ptr, gr.ptr, gw.ptr, None, EPS, None, y1.ptr, m.ptr, s.ptr)
    assert np.abs(y.numpy() - (y1.numpy() + b)).max() <= 4 * F32 * (np.abs(y.numpy()).max() + np.abs(b).max())
    ws = hip.Buffer(hip.lib().mle_add_layernorm_ws_bytes(40, 200))
    outs = []
    for dw, db in ((1, 1), (1, 0), (0, 1), (0, 0)):
        d, gw1, gb1 = hip.Buffer.empty(n), hip.Buffer.zeros(200), hip.Buffer.zeros(200)
        hip.call("mle_add_layernorm_bwd", None, 40, 200, h.ptr, gw.ptr, m.ptr, s.ptr, gdy.ptr, None, d.ptr, 0,
                 gw1.ptr if dw else None, gb1.ptr if db else None, 0, ws.ptr if dw or db else None, ws.nbytes if dw or db else 0)
        outs.append((d.numpy(), gw1.numpy(), gb1.numpy()))
    for d, a, c in outs[1:]:
        assert np.array_equal(d, outs[0][0])
    assert np.array_equal(outs[1][1], outs[0][1]) and np.array_equal(outs[2][2], outs[0][2])
    assert (outs[1][2] == 0).all() and (outs[2][1] == 0).all()


@pytest.mark.parametrize("rows,cols", [(12, 300), (6, 4000), (4, 9000), (250, 700)])
def test_in_place(hip, rows, cols):
    """h over x, and dh over dy, give what buffers of their own give."""
    r = rng(4)
    x, res, dy = (r.standard_normal((rows, cols)).astype(np.float32) for _ in range(3))
    ws = hip.Buffer(hip.lib().mle_add_layernorm_ws_bytes(rows, cols))
    out = []
    for own in (True, False):
        gx, gr, gdy = (hip.Buffer.from_array(a) for a in (x, res, dy))
        gh = hip.Buffer.empty((rows, cols)) if own else gx
        gdh = hip.Buffer.empty((rows, cols)) if own else gdy
        gy, gm, gs, dw, db = (hip.Buffer.empty(n) for n in ((rows, cols), rows, rows, cols, cols))
        hip.call("mle_add_layernorm_fwd", None, rows, cols, gx.ptr, gr.ptr, None, None, EPS, gh.ptr, gy.ptr, gm.ptr, gs.ptr)
        hip.call("mle_add_layernorm_bwd", None, rows, cols, gh.ptr, None, gm.ptr, gs.ptr, gdy.ptr, None, gdh.ptr, 0, dw.ptr,
                 db.ptr, 0, ws.ptr, ws.nbytes)
        out.append([b.numpy() for b in (gh, gy, gm, gs, gdh, dw, db)])
    for a, b in zip(*out):
        assert np.array_equal(a, b)


def test_even_rows_and_not_finite(hip):
    x = rng(5).standard_normal((5, 70)).astype(np.float32)
    x[1], x[2, 3], x[3, 60] = 4.0, np.nan, np.inf
    gx, gy, gm, gs = hip.Buffer.from_array(x), hip.Buffer.empty((5, 70)), hip.Buffer.empty(5), hip.Buffer.empty(5)
    hip.call("mle_add_layernorm_fwd", None, 5, 70, gx.ptr, None, None, None, EPS, None, gy.ptr, gm.ptr, gs.ptr)
    y = gy.numpy()
    assert (y[1] == 0).all() and np.isnan(y[2]).all() and np.isnan(y[3]).all() and np.isfinite(y[[0, 4]]).all()
    hip.call("mle_add_layernorm_fwd", None, 0, 70, None, None, None, None, EPS, None, None, None, None)
    for acc in (1, 0):
        dw, db = (hip.Buffer.from_array(np.ones(70, np.float32)) for _ in range(2))
        hip.call("mle_add_layernorm_bwd", None, 0, 70, None, None, None, None, None, None, None, 0, dw.ptr, db.ptr, acc, None, 0)
        assert (dw.numpy() == acc).all() and (db.numpy() == acc).all()


def test_gradient_against_differences(hip):
    """dh, dw and db against central differences of <y, dy> of the 64-bit formula."""
    r = rng(6)
    rows, cols = 3, 40
    x, dy = r.standard_normal((rows, cols)).astype(np.float32), r.standard_normal((rows, cols)).astype(np.float32)
    w, b = (1 + 0.2 * r.standard_normal(cols)).astype(np.float32), r.standard_normal(cols).astype(np.float32)
    gx, gw, gb, gdy = (hip.Buffer.from_array(a) for a in (x, w, b, dy))
    gm, gs, dh, dw, db = (hip.Buffer.empty(n) for n in (rows, rows, (rows, cols), cols, cols))
    ws = hip.Buffer(hip.lib().mle_add_layernorm_ws_bytes(rows, cols))
    hip.call("mle_add_layernorm_fwd", None, rows, cols, gx.ptr, None, gw.ptr, gb.ptr, EPS, None, None, gm.ptr, gs.ptr)
    hip.call("mle_add_layernorm_bwd", None, rows, cols, gx.ptr, gw.ptr, gm.ptr, gs.ptr, gdy.ptr, None, dh.ptr, 0, dw.ptr, db.ptr,
             0, ws.ptr, ws.nbytes)

    def f(h, v, c):
        return float(((norm64(h)[2] * v + c) * dy).sum())

    args, step = [a.astype(np.float64) for a in (x, w, b)], 1e-5
    for k, (got, places) in enumerate(((dh, [(0, 0), (1, 17), (2, 39)]), (dw, [0, 21, 39]), (db, [0, 5, 39]))):
        for p in places:
            y = [a.copy() for a in args]
            y[k][p] += step
            up = f(*y)
            y[k][p] -= 2 * step
            assert abs((up - f(*y)) / (2 * step) - got.numpy()[p]) <= 1e-5
