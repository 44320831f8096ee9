"""The layer norm's backward of rows whose mean lies far above their spread: what the differences
within a row hold, dh, dw and db keep, at the sizes where it changes form.  And of the widest rows."""
import numpy as np
import pytest

from conftest import rng

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -24  # half a step of fp32
EPS = 1e-12       # (far below the rows' spread)


def data(rows, cols):
    """Every third row an ordinary one, the others near 1000 with differences of some 0.01."""
    r = rng(rows + cols)
    x = (1000 * r.choice([-1, 1], (rows, 1)) + 0.01 * r.standard_normal((rows, cols))).astype(np.float32)
    x[::3] = r.standard_normal(x[::3].shape)
    w, b = (1 + 0.2 * r.standard_normal(cols)).astype(np.float32), r.standard_normal(cols).astype(np.float32)
    dy, dres = (r.standard_normal((rows, cols)).astype(np.float32) for _ in range(2))
    return x, w, b, dy, dres


def run(hip, rows, cols, x, w, b, dy, dres, in_place=False, sums=True):
    gx, gw, gb, gdy, gdr = (hip.Buffer.from_array(a) for a in (x, w, b, dy, dres))
    gm, gs, y, dw, db = (hip.Buffer.empty(n) for n in (rows, rows, (rows, cols), cols, cols))
    dh = gdy if in_place else hip.Buffer.empty((rows, cols))
    ws = hip.Buffer(hip.lib().mle_add_layernorm_ws_bytes(rows, cols))
    hip.call("mle_add_layernorm_fwd", None, rows, cols, gx.ptr, None, gw.ptr, gb.ptr, EPS, None, y.ptr, gm.ptr, gs.ptr)
    hip.call("mle_add_layernorm_bwd", None, rows, cols, gx.ptr, gw.ptr, gm.ptr, gs.ptr, gdy.ptr, gdr.ptr, dh.ptr, 0,
             dw.ptr if sums else None, db.ptr if sums else None, 0, ws.ptr if sums else None, ws.nbytes if sums else 0)
    hip.sync()
    return [t.numpy() for t in (y, dh, dw, db)]


@pytest.mark.parametrize("rows,cols", [(1, 40), (40, 200), (60, 700), (256, 1500), (257, 700), (700, 300), (300, 2000), (20, 3000),
                                       (9, 7001), (6, 9000), (700, 8200)])
def test_gradients_of_rows_far_from_zero(hip, rows, cols):
    x, w, b, dy, dres = data(rows, cols)
    y, dh, dw, db = run(hip, rows, cols, x, w, b, dy, dres)
    h = x.astype(np.float64)
    mean = h.mean(1, keepdims=True)
    rstd = 1 / np.sqrt(((h - mean) ** 2).mean(1, keepdims=True) + float(np.float32(EPS)))
    u = (h - mean) * rstd
    g = dy * w.astype(np.float64)
    m1, m2 = g.mean(1, keepdims=True), (g * u).mean(1, keepdims=True)
    # u: h - mean, the rest of the mean, rstd and their product round; an ordinary row's mean (its
    # rest left out below 4 spreads) moves u by 2^-22 at most
    eu = F32 * (5 * np.abs(u) + np.where(np.abs(mean) * rstd > 4, 1, 4))
    size = rstd * (np.abs(g) + np.abs(g).mean(1, keepdims=True) + np.abs(u) * np.abs(g * u).mean(1, keepdims=True))
    spill = rstd * (eu * np.abs(g * u).mean(1, keepdims=True) + np.abs(u) * (np.abs(g) * eu).mean(1, keepdims=True))
    assert (np.abs(dh - (rstd * (g - m1 - u * m2) + dres)) <= 12 * F32 * (size + np.abs(dres)) + 2 * spill).all()
    want = (dy * u).sum(0)
    assert (np.abs(dw - want) <= F32 * (rows + 8) * np.abs(dy * u).sum(0) + (np.abs(dy) * eu).sum(0)).all()
    assert (np.abs(db - dy.astype(np.float64).sum(0)) <= F32 * (rows + 8) * np.abs(dy).sum(0)).all()


@pytest.mark.parametrize("rows,cols", [(60, 700), (250, 2048), (300, 500), (20, 3000), (6, 9000)])
def test_forms_agree(hip, rows, cols):
    """Over dy in place, and without the weight's sums, the same bits."""
    x, w, b, dy, dres = data(rows, cols)
    one = run(hip, rows, cols, x, w, b, dy, dres)
    two = run(hip, rows, cols, x, w, b, dy, dres, in_place=True)
    for a, c in zip(one, two):
        assert np.array_equal(a, c)
    assert np.array_equal(one[1], run(hip, rows, cols, x, w, b, dy, dres, sums=False)[1])


def test_more_columns_than_a_join_takes(hip):
    """A row of 2^26 + 5 values: 64 threads to each column are more than a launch has."""
    cols = (1 << 26) + 5
    r = rng(3)
    x, dy = (r.standard_normal((1, cols), dtype=np.float32) for _ in range(2))
    gx, gdy, gm, gs, dw = hip.Buffer.from_array(x), hip.Buffer.from_array(dy), hip.Buffer.empty(1), hip.Buffer.empty(1), hip.Buffer.empty(cols)
    db, ws = hip.Buffer.from_array(np.full(cols, 7, np.float32)), hip.Buffer(hip.lib().mle_add_layernorm_ws_bytes(1, cols))
    hip.call("mle_add_layernorm_fwd", None, 1, cols, gx.ptr, None, None, None, EPS, None, None, gm.ptr, gs.ptr)
    hip.call("mle_add_layernorm_bwd", None, 1, cols, gx.ptr, None, gm.ptr, gs.ptr, gdy.ptr, None, gdy.ptr, 0, dw.ptr, db.ptr, 0, ws.ptr,
             ws.nbytes)
    hip.sync()
    h = x[0].astype(np.float64)
    u = (h - h.mean()) / np.sqrt(h.var() + float(np.float32(EPS)))
    # the mean's rounding, h - mean, rstd and two products
    assert (np.abs(dw.numpy() - dy[0] * u) <= F32 * np.abs(dy[0]) * (6 * np.abs(u) + 1)).all()
    assert np.array_equal(db.numpy(), dy[0])
