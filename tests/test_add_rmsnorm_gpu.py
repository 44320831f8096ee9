"""The residual Add with the root-mean-square norm against 64 bits; the 8 bits
against the format in numpy."""
import numpy as np
import pytest

import q8_ref
from conftest import rng

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -24  # half a step of fp32
EPS = 1e-5


def at(hip, a, shift):
    """A device copy of a that begins `shift` floats into its buffer."""
    b = hip.Buffer.from_array(np.concatenate([np.zeros(shift, np.float32), a.reshape(-1).astype(np.float32)]))
    return b, b.ptr + 4 * shift


SHAPES = [(1, 1), (1, 32), (3, 31), (5, 33), (64, 256), (7, 330), (130, 512), (9, 1000), (33, 1024), (6, 1500), (40, 2048),
          (3, 2052), (5, 4096), (2, 6001), (3, 8192), (2, 8200), (3, 20001), (1500, 64),
          (4, 7), (6, 37), (3, 38), (5, 2049), (2, 8191)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("residual,weight,acc,shift", [(1, 1, 0, 0), (0, 1, 1, 0), (1, 0, 1, 1)])
def test_forward_and_backward(hip, rows, cols, residual, weight, acc, shift):
    r = rng(rows * 31 + cols)
    x, res, dy, dres = (r.standard_normal((rows, cols)).astype(np.float32) for _ in range(4))
    w = (1 + 0.2 * r.standard_normal(cols)).astype(np.float32)
    old_dh, old_dw = r.standard_normal((rows, cols)).astype(np.float32), r.standard_normal(cols).astype(np.float32)
    ng, ldq = -(-cols // 32), cols + 3 * shift
    bx, px = at(hip, x, shift)
    br, pr = at(hip, res, shift)
    bw, pw = at(hip, w, shift)
    bh, ph = at(hip, np.zeros((rows, cols)), shift)
    by, py = at(hip, np.zeros((rows, cols)), shift)
    gs, gq, ge = hip.Buffer.empty(rows), hip.Buffer.empty((rows, ldq), np.int8), hip.Buffer.empty((rows, ng), np.uint8)
    hip.call("mle_add_rmsnorm_q8_fwd", None, rows, cols, px, pr if residual else None, pw if weight else None, EPS, ph, py,
             gs.ptr, gq.ptr, ldq, ge.ptr, ng)
    h = bh.numpy().reshape(-1)[shift:].reshape(rows, cols)
    y = by.numpy().reshape(-1)[shift:].reshape(rows, cols)
    assert np.array_equal(h, x + res if residual else x)
    h64 = h.astype(np.float64)
    w64 = w.astype(np.float64) if weight else np.ones(cols)
    s = 1 / np.sqrt((h64 ** 2).mean(1, keepdims=True) + np.float64(np.float32(EPS)))
    ref = h64 * s * w64
    assert (np.abs(y - ref) <= F32 * (1 + 1e-6) * np.abs(ref) + 2.0 ** -149).all()  # rounded once
    assert (np.abs(gs.numpy() - s[:, 0]) <= F32 * (1 + 1e-6) * s[:, 0]).all()
    q, e = q8_ref.quantize(y)
    assert np.array_equal(gq.numpy()[:, :cols], q) and np.array_equal(ge.numpy(), e)

    bdy, pdy = at(hip, dy, shift)
    bdr, pdr = at(hip, dres, shift)
    bdh, pdh = at(hip, old_dh, shift)
    gdw = hip.Buffer.from_array(old_dw)
    ws = hip.Buffer(hip.lib().mle_add_rmsnorm_ws_bytes(rows, cols))
    hip.call("mle_add_rmsnorm_bwd", None, rows, cols, ph, pw if weight else None, gs.ptr, pdy, pdr if residual else None, pdh,
             acc, gdw.ptr, acc, ws.ptr, ws.nbytes)
    u, g = h64 * s, dy.astype(np.float64) * w64
    m = (g * u).mean(1, keepdims=True)
    dh = s * (g - u * m) + (dres if residual else 0) + (old_dh if acc else 0)
    got = bdh.numpy().reshape(-1)[shift:].reshape(rows, cols)
    # s, u, g, g u, u m, the difference, the product and the two sums round once
    # each; the mean's own rounding and its factors' give six more
    size = s * (np.abs(g) + np.abs(u) * np.abs(g * u).mean(1, keepdims=True)) + np.abs(dres) + np.abs(old_dh)
    assert (np.abs(got - dh) <= 16 * F32 * size).all()
    dw = (dy * u).sum(0) + (old_dw if acc else 0)
    assert (np.abs(gdw.numpy() - dw) <= F32 * ((rows + 8) * np.abs(dy * u).sum(0) + 2 * np.abs(old_dw))).all()


def test_optional_outputs(hip):
    """h, y, the 8 bits and dw can each be left out; what stays is the same."""
    r = rng(2)
    x, res, dy = (r.standard_normal((40, 200)).astype(np.float32) for _ in range(3))
    gx, gr, gdy = (hip.Buffer.from_array(a) for a in (x, res, dy))
    full = [hip.Buffer.empty((40, 200)), hip.Buffer.empty((40, 200)), hip.Buffer.empty((40, 200), np.int8),
            hip.Buffer.empty((40, 7), np.uint8), hip.Buffer.empty(40)]
    hip.call("mle_add_rmsnorm_q8_fwd", None, 40, 200, gx.ptr, gr.ptr, None, EPS, full[0].ptr, full[1].ptr, full[4].ptr,
             full[2].ptr, 200, full[3].ptr, 7)
    h, y, q, e, s = (b.numpy() for b in full)
    one = [hip.Buffer.empty((40, 200)), hip.Buffer.empty((40, 200)), hip.Buffer.empty((40, 200), np.int8),
           hip.Buffer.empty((40, 7), np.uint8), hip.Buffer.empty(40)]
    hip.call("mle_add_rmsnorm_q8_fwd", None, 40, 200, gx.ptr, gr.ptr, None, EPS, None, one[1].ptr, one[4].ptr, None, 0, None, 0)
    assert np.array_equal(one[1].numpy(), y) and np.array_equal(one[4].numpy(), s)
    hip.call("mle_add_rmsnorm_q8_fwd", None, 40, 200, gx.ptr, gr.ptr, None, EPS, None, None, one[4].ptr, one[2].ptr, 200,
             one[3].ptr, 7)
    assert np.array_equal(one[2].numpy(), q) and np.array_equal(one[3].numpy(), e)
    a, b, dw = hip.Buffer.empty((40, 200)), hip.Buffer.empty((40, 200)), hip.Buffer.empty(200)
    ws = hip.Buffer(hip.lib().mle_add_rmsnorm_ws_bytes(40, 200))
    hip.call("mle_add_rmsnorm_bwd", None, 40, 200, full[0].ptr, None, full[4].ptr, gdy.ptr, None, a.ptr, 0, dw.ptr, 0, ws.ptr,
             ws.nbytes)
    hip.call("mle_add_rmsnorm_bwd", None, 40, 200, full[0].ptr, None, full[4].ptr, gdy.ptr, None, b.ptr, 0, None, 0, None, 0)
    assert np.array_equal(a.numpy(), b.numpy())


@pytest.mark.parametrize("rows,cols", [(12, 300), (6, 3000), (4, 9000)])
def test_in_place(hip, rows, cols):
    """h over x, and dh over dy, give what buffers of their own give."""
    r = rng(4)
    x, res, dy = (r.standard_normal((rows, cols)).astype(np.float32) for _ in range(3))
    ws = hip.Buffer(hip.lib().mle_add_rmsnorm_ws_bytes(rows, cols))
    out = []
    for own in (True, False):
        gx, gr, gdy = (hip.Buffer.from_array(a) for a in (x, res, dy))
        gh = hip.Buffer.empty((rows, cols)) if own else gx
        gdh = hip.Buffer.empty((rows, cols)) if own else gdy
        gy, gs, dw = hip.Buffer.empty((rows, cols)), hip.Buffer.empty(rows), hip.Buffer.empty(cols)
        hip.call("mle_add_rmsnorm_q8_fwd", None, rows, cols, gx.ptr, gr.ptr, None, EPS, gh.ptr, gy.ptr, gs.ptr, None, 0, None,
                 0)
        hip.call("mle_add_rmsnorm_bwd", None, rows, cols, gh.ptr, None, gs.ptr, gdy.ptr, None, gdh.ptr, 0, dw.ptr, 0, ws.ptr,
                 ws.nbytes)
        out.append([b.numpy() for b in (gh, gy, gs, gdh, dw)])
    for a, b in zip(*out):
        assert np.array_equal(a, b)


def test_zero_rows_and_not_finite(hip):
    x = rng(5).standard_normal((5, 70)).astype(np.float32)
    x[1], x[2, 3], x[3, 60] = 0.0, np.nan, np.inf
    gx, gy, gs = hip.Buffer.from_array(x), hip.Buffer.empty((5, 70)), hip.Buffer.empty(5)
    gq, ge = hip.Buffer.empty((5, 70), np.int8), hip.Buffer.empty((5, 3), np.uint8)
    hip.call("mle_add_rmsnorm_q8_fwd", None, 5, 70, gx.ptr, None, None, EPS, None, gy.ptr, gs.ptr, gq.ptr, 70, ge.ptr, 3)
    y = gy.numpy()
    assert (y[1] == 0).all() and np.isnan(y[2]).all() and np.isnan(y[3, 60]) and np.isfinite(y[[0, 4]]).all()
    q, e = q8_ref.quantize(y)
    assert np.array_equal(gq.numpy(), q) and np.array_equal(ge.numpy(), e)
    hip.call("mle_add_rmsnorm_q8_fwd", None, 0, 70, None, None, None, EPS, None, None, None, None, 0, None, 0)
    dw = hip.Buffer.from_array(np.ones(70, np.float32))
    hip.call("mle_add_rmsnorm_bwd", None, 0, 70, None, None, None, None, None, None, 0, dw.ptr, 1, None, 0)
    assert (dw.numpy() == 1).all()
    hip.call("mle_add_rmsnorm_bwd", None, 0, 70, None, None, None, None, None, None, 0, dw.ptr, 0, None, 0)
    assert (dw.numpy() == 0).all()


def test_gradient_against_differences(hip):
    """dh and dw against central differences of <y, dy> of the 64-bit formula."""
    r = rng(6)
    rows, cols = 3, 40
    x, dy = r.standard_normal((rows, cols)).astype(np.float32), r.standard_normal((rows, cols)).astype(np.float32)
    w = (1 + 0.2 * r.standard_normal(cols)).astype(np.float32)
    gx, gw, gdy, gs = (hip.Buffer.from_array(a) for a in (x, w, dy, np.zeros(rows, np.float32)))
    dh, dw = hip.Buffer.empty((rows, cols)), hip.Buffer.empty(cols)
    ws = hip.Buffer(hip.lib().mle_add_rmsnorm_ws_bytes(rows, cols))
    hip.call("mle_add_rmsnorm_q8_fwd", None, rows, cols, gx.ptr, None, gw.ptr, EPS, None, None, gs.ptr, None, 0, None, 0)
    hip.call("mle_add_rmsnorm_bwd", None, rows, cols, gx.ptr, gw.ptr, gs.ptr, gdy.ptr, None, dh.ptr, 0, dw.ptr, 0, ws.ptr,
             ws.nbytes)

    def f(h, v):
        return float((h / np.sqrt((h * h).mean(1, keepdims=True) + EPS) * v * dy).sum())

    h64, w64, step = x.astype(np.float64), w.astype(np.float64), 1e-5
    for i, j in [(0, 0), (1, 17), (2, 39)]:
        d = np.zeros_like(h64)
        d[i, j] = step
        assert abs((f(h64 + d, w64) - f(h64 - d, w64)) / (2 * step) - dh.numpy()[i, j]) <= 1e-5
    for j in (0, 21, 39):
        d = np.zeros_like(w64)
        d[j] = step
        assert abs((f(h64, w64 + d) - f(h64, w64 - d)) / (2 * step) - dw.numpy()[j]) <= 1e-5
