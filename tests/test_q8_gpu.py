"""Activations kept in 8 bits against numpy (the format is exact, so codes and
values are equal bit for bit) and against 64 bits."""
import math

import numpy as np
import pytest

import q8_ref
from conftest import rng

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -24  # half a step of fp32


def padded(a, ld, fill):
    """A device copy of a with rows of ld elements, the rest `fill`."""
    full = np.full((a.shape[0], ld), fill, dtype=a.dtype)
    full[:, : a.shape[1]] = a
    return full


def quantize(hip, x, ldx, ldq, lde):
    rows, cols = x.shape
    gx = hip.Buffer.from_array(padded(x, ldx, 7.0))
    gq = hip.Buffer.from_array(np.full((rows, ldq), 99, dtype=np.int8))
    ge = hip.Buffer.from_array(np.full((rows, lde), 77, dtype=np.uint8))
    hip.call("mle_q8_quantize", None, rows, cols, gx.ptr, ldx, gq.ptr, ldq, ge.ptr, lde)
    return gx, gq, ge


def samples(r, rows, cols):
    x = (r.standard_normal((rows, cols)) * np.exp2(r.integers(-20, 20, (rows, 1)))).astype(np.float32)
    x[0] = 0.0
    if rows > 3:
        x[1] = np.float32(2.0) ** -140          # a group below the smallest step
        x[2] = (r.integers(-255, 256, cols) / 2).astype(np.float32)  # ties, and 127.5 itself
        x[3, : min(cols, 4)] = [3.4e38, -3.4e38, 1e-45, 127.5][: min(cols, 4)]
    return x


@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (4, 32, 0), (5, 31, 1), (7, 33, 2), (64, 96, 8), (37, 330, 3),
                                           (3, 4096, 0), (300, 129, 0), (1, 2048, 4), (5, 34, 0), (6, 35, 1), (5, 36, 0),
                                           (7, 37, 0), (4, 38, 5), (9, 39, 0), (2, 7, 0)])
def test_quantize_and_back(hip, rows, cols, pad):
    x = samples(rng(rows * 1000 + cols), rows, cols)
    ng = -(-cols // 32)
    _, gq, ge = quantize(hip, x, cols + pad, cols + pad, ng + pad)
    q, e = q8_ref.quantize(x)
    got_q, got_e = gq.numpy(), ge.numpy()
    assert np.array_equal(got_q[:, :cols], q) and (got_q[:, cols:] == 99).all()
    assert np.array_equal(got_e[:, :ng], e) and (got_e[:, ng:] == 77).all()
    gy = hip.Buffer.from_array(np.full((rows, cols + pad), 5.0, dtype=np.float32))
    hip.call("mle_q8_dequantize", None, rows, cols, gq.ptr, cols + pad, ge.ptr, ng + pad, gy.ptr, cols + pad)
    y = gy.numpy()
    assert np.array_equal(y[:, :cols], q8_ref.values(q, e)) and (y[:, cols:] == 5.0).all()
    step = np.ldexp(1.0, e.astype(int) - 127)[:, np.arange(cols) // 32]
    # half a step; from 127.5 * 2^121 up the nearest multiple of that step is 2^128,
    # which is no float, so 127 steps stand for values below 128 steps
    most = np.where(np.abs(x.astype(np.float64)) >= 127.5 * 2.0 ** 121, step, step / 2)
    assert (np.abs(y[:, :cols].astype(np.float64) - x) <= most).all()


def test_quantize_not_finite(hip):
    x = rng(3).standard_normal((4, 96)).astype(np.float32)
    x[0, 40], x[1, 3], x[2, 70], x[2, 71] = np.nan, np.inf, -np.inf, np.inf
    _, gq, ge = quantize(hip, x, 96, 96, 3)
    q, e = q8_ref.quantize(x)
    assert np.array_equal(gq.numpy(), q) and np.array_equal(ge.numpy(), e)
    gy = hip.Buffer.empty((4, 96))
    hip.call("mle_q8_dequantize", None, 4, 96, gq.ptr, 96, ge.ptr, 3, gy.ptr, 96)
    y = gy.numpy()
    assert np.isnan(y[0, 32:64]).all() and np.isfinite(y[0, :32]).all() and np.isfinite(y[0, 64:]).all()
    assert y[1, 3] == np.inf and y[2, 70] == -np.inf and y[2, 71] == np.inf and np.isfinite(y[3]).all()


def act64(kind, x):
    if kind == "relu":
        return np.maximum(x, 0)
    if kind == "silu":
        return x / (1 + np.exp(-x))
    return 0.5 * x * (1 + np.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))


def act_grad64(kind, x):
    if kind == "relu":
        return (x > 0).astype(np.float64)
    if kind == "silu":
        s = 1 / (1 + np.exp(-x))
        return s * (1 + x * (1 - s))
    t = np.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3))
    return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 0.134145 * x * x)


@pytest.mark.parametrize("kind", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("rows,cols,pad,acc", [(1, 1, 0, 0), (33, 70, 2, 1), (64, 256, 0, 0), (20, 330, 0, 1)])
def test_act(hip, kind, rows, cols, pad, acc):
    r = rng(cols)
    x = (r.standard_normal((rows, cols)) * 2).astype(np.float32)
    dy, old = (r.standard_normal((rows, cols)).astype(np.float32) for _ in range(2))
    ld, ng = cols + pad, -(-cols // 32)
    gx, gy = hip.Buffer.from_array(padded(x, ld, 7.0)), hip.Buffer.from_array(np.full((rows, ld), 5, np.float32))
    gq, ge = hip.Buffer.empty((rows, ld), np.int8), hip.Buffer.empty((rows, ng), np.uint8)
    hip.call("mle_q8_act_fwd", None, hip.ACT[kind], rows, cols, gx.ptr, ld, gy.ptr, ld, gq.ptr, ld, ge.ptr, ng)
    q, e = q8_ref.quantize(x)
    assert np.array_equal(gq.numpy()[:, :cols], q) and np.array_equal(ge.numpy(), e)
    y = gy.numpy()
    # about ten roundings and two library functions of a few steps each, of
    # terms no larger than |x| + 1
    assert (np.abs(y[:, :cols] - act64(kind, x.astype(np.float64))) <= 32 * F32 * (np.abs(x) + 1)).all()
    assert (y[:, cols:] == 5).all()
    # the elementwise forward gives the same bits
    fx, fy = hip.Buffer.from_array(x), hip.Buffer.empty((rows, cols))
    hip.call("mle_act_fwd", None, hip.ACT[kind], fx.ptr, fy.ptr, rows * cols)
    assert np.array_equal(fy.numpy(), y[:, :cols])
    gdy, gdx = hip.Buffer.from_array(padded(dy, ld, 7.0)), hip.Buffer.from_array(padded(old, ld, 3.0))
    hip.call("mle_q8_act_bwd", None, hip.ACT[kind], rows, cols, gq.ptr, ld, ge.ptr, ng, gdy.ptr, ld, gdx.ptr, ld, acc)
    dx, v = gdx.numpy(), q8_ref.values(q, e).astype(np.float64)
    ref = act_grad64(kind, v) * dy + (old if acc else 0)
    # the derivative's terms reach |x|^3 du before they cancel against 1 - tanh^2
    assert (np.abs(dx[:, :cols] - ref) <= F32 * (64 * (1 + v * v) * np.abs(dy) + 2 * np.abs(old))).all()
    assert (dx[:, cols:] == 3).all()
    # the elementwise backward on the kept values gives the same bits
    fv, fdy, fdx = hip.Buffer.from_array(v.astype(np.float32)), hip.Buffer.from_array(dy), hip.Buffer.from_array(old)
    hip.call("mle_act_bwd", None, hip.ACT[kind], fv.ptr, fdy.ptr, fdx.ptr, rows * cols, acc)
    assert np.array_equal(fdx.numpy(), dx[:, :cols])


def test_act_in_place(hip):
    r = rng(8)
    x, dy = (r.standard_normal((50, 64)).astype(np.float32) for _ in range(2))
    gx, gdy = hip.Buffer.from_array(x), hip.Buffer.from_array(dy)
    gq, ge = hip.Buffer.empty((50, 64), np.int8), hip.Buffer.empty((50, 2), np.uint8)
    hip.call("mle_q8_act_fwd", None, hip.ACT["silu"], 50, 64, gx.ptr, 64, gx.ptr, 64, gq.ptr, 64, ge.ptr, 2)
    hip.call("mle_q8_act_bwd", None, hip.ACT["silu"], 50, 64, gq.ptr, 64, ge.ptr, 2, gdy.ptr, 64, gdy.ptr, 64, 0)
    assert np.array_equal(gq.numpy(), q8_ref.quantize(x)[0])
    assert np.allclose(gx.numpy(), act64("silu", x.astype(np.float64)), rtol=1e-6, atol=1e-6)
    assert np.allclose(gdy.numpy(), act_grad64("silu", q8_ref.kept(x).astype(np.float64)) * dy, rtol=1e-5, atol=1e-6)


def wgrad(hip, x, dy, ldq, lde, lddy, lddw, old_dw, old_db, acc, bias=True):
    rows, inp = x.shape
    out = dy.shape[1]
    q, e = q8_ref.quantize(x)
    gq, ge = hip.Buffer.from_array(padded(q, ldq, 99)), hip.Buffer.from_array(padded(e, lde, 200))
    gdy, gdw = hip.Buffer.from_array(padded(dy, lddy, 1e30)), hip.Buffer.from_array(padded(old_dw, lddw, 5.0))
    gdb = hip.Buffer.from_array(old_db)
    ws = hip.Buffer(hip.lib().mle_q8_linear_wgrad_ws_bytes(rows, inp, out))
    hip.call("mle_q8_linear_wgrad", None, rows, inp, out, gq.ptr, ldq, ge.ptr, lde, gdy.ptr, lddy, gdw.ptr, lddw,
             gdb.ptr if bias else None, acc, ws.ptr, ws.nbytes)
    return gdw.numpy(), gdb.numpy()


@pytest.mark.parametrize("rows,inp,out,pad,acc", [(1, 1, 1, 0, 0), (1, 40, 24, 1, 1), (31, 33, 65, 3, 0), (64, 64, 64, 0, 1),
                                                  (200, 96, 130, 0, 0), (1000, 330, 516, 0, 0), (257, 128, 256, 8, 1),
                                                  (2048, 256, 384, 0, 0), (4096, 48, 52, 0, 0), (333, 1024, 64, 0, 0),
                                                  (500, 3, 130, 0, 1), (70, 5, 9, 2, 0), (1500, 700, 2100, 0, 0),
                                                  (8200, 257, 1030, 1, 1)])
def test_linear_wgrad(hip, rows, inp, out, pad, acc):
    r = rng(rows + inp + out)
    x = (r.standard_normal((rows, inp)) * np.exp2(r.integers(-6, 6, (rows, 1)))).astype(np.float32)
    dy = (r.standard_normal((rows, out)) * np.exp2(r.integers(-10, 2, (1, out)))).astype(np.float32)
    old_dw, old_db = r.standard_normal((inp, out)).astype(np.float32), r.standard_normal(out).astype(np.float32)
    got, db = wgrad(hip, x, dy, inp + pad, -(-inp // 32) + pad, out + pad, out + pad, old_dw, old_db, acc)
    v, d = q8_ref.kept(x).astype(np.float64), dy.astype(np.float64)
    ref = v.T @ d + (old_dw if acc else 0)
    # a sum of `rows` products in fp32, truncated or rounded: a step each at most
    tol = 2 * F32 * ((rows + 4) * (np.abs(v).T @ np.abs(d)) + 2 * np.abs(old_dw))
    assert (np.abs(got[:, :out] - ref) <= tol).all()
    assert (got[:, out:] == 5.0).all()
    ref_db = d.sum(0) + (old_db if acc else 0)
    assert (np.abs(db - ref_db) <= 2 * F32 * ((rows + 4) * np.abs(d).sum(0) + 2 * np.abs(old_db))).all()


def test_linear_wgrad_accuracy(hip):
    """As exact as fp32 products of the kept values: the 2-norm error stays below
    that of rounding each product once."""
    r = rng(5)
    x = np.maximum(r.standard_normal((4096, 256)), 0).astype(np.float32)
    dy = r.standard_normal((4096, 320)).astype(np.float32)
    got, _ = wgrad(hip, x, dy, 256, 8, 320, 320, np.zeros((256, 320), np.float32), np.zeros(320, np.float32), 0)
    ref = q8_ref.kept(x).astype(np.float64).T @ dy.astype(np.float64)
    assert np.linalg.norm(got - ref) <= 1e-6 * np.linalg.norm(ref)


def test_linear_wgrad_without_bias_and_rows(hip):
    r = rng(6)
    x, dy = r.standard_normal((96, 64)).astype(np.float32), r.standard_normal((96, 32)).astype(np.float32)
    zero, kept_db = np.zeros((64, 32), np.float32), np.full(32, 9.0, np.float32)
    got, db = wgrad(hip, x, dy, 64, 2, 32, 32, zero, kept_db, 0, bias=False)
    assert np.allclose(got, q8_ref.kept(x).T @ dy, rtol=1e-4, atol=1e-4) and (db == 9.0).all()
    gdw, gdb = hip.Buffer.from_array(zero + 3), hip.Buffer.from_array(kept_db)
    hip.call("mle_q8_linear_wgrad", None, 0, 64, 32, None, 64, None, 2, None, 32, gdw.ptr, 32, gdb.ptr, 1, None, 0)
    assert (gdw.numpy() == 3).all() and (gdb.numpy() == 9).all()
    hip.call("mle_q8_linear_wgrad", None, 0, 64, 32, None, 64, None, 2, None, 32, gdw.ptr, 32, gdb.ptr, 0, None, 0)
    assert (gdw.numpy() == 0).all() and (gdb.numpy() == 0).all()


@pytest.mark.parametrize("scale", [2.0 ** -120, 2.0 ** 60])
def test_linear_wgrad_extreme_values(hip, scale):
    r = rng(7)
    x = (r.standard_normal((128, 64)) * scale).astype(np.float32)
    dy = (r.standard_normal((128, 64)) * min(1.0, 1 / scale)).astype(np.float32)
    got, _ = wgrad(hip, x, dy, 64, 2, 64, 64, np.zeros((64, 64), np.float32), np.zeros(64, np.float32), 0)
    v, d = q8_ref.kept(x).astype(np.float64), dy.astype(np.float64)
    assert (np.abs(got - v.T @ d) <= 2 * F32 * 132 * (np.abs(v).T @ np.abs(d)) + 2.0 ** -149).all()


def test_linear_wgrad_not_finite_stays_in_its_column(hip):
    """A NaN among the kept values reaches its group's rows of dW alone."""
    r = rng(9)
    x, dy = r.standard_normal((100, 96)).astype(np.float32), r.standard_normal((100, 40)).astype(np.float32)
    x[17, 40] = np.nan
    got, db = wgrad(hip, x, dy, 96, 3, 40, 40, np.zeros((96, 40), np.float32), np.zeros(40, np.float32), 0)
    assert np.isnan(got[32:64]).all() and np.isfinite(got[:32]).all() and np.isfinite(got[64:]).all()
    assert np.isfinite(db).all()


def test_linear_wgrad_repeats(hip):
    r = rng(10)
    x, dy = r.standard_normal((3000, 200)).astype(np.float32), r.standard_normal((3000, 136)).astype(np.float32)
    a = [wgrad(hip, x, dy, 200, 7, 136, 136, np.zeros((200, 136), np.float32), np.zeros(136, np.float32), 0) for _ in range(2)]
    assert np.array_equal(a[0][0], a[1][0]) and np.array_equal(a[0][1], a[1][1])


# (rows, in, out): few rows, so that the bound of their sums is tight; the narrow, the
# small and the large tile, then row splits
GRADIENT_SHAPES = [(8, 3, 130), (8, 64, 64), (16, 300, 40), (8, 2048, 2048), (4096, 48, 52)]


@pytest.mark.parametrize("rows,inp,out", GRADIENT_SHAPES)
@pytest.mark.parametrize("xs,ds", [(0, -112), (0, -117), (0, -122), (24, -130), (30, -140), (60, 55), (0, 118), (-100, 120)])
def test_linear_wgrad_over_the_range_of_dy(hip, rows, inp, out, xs, ds):
    """Gradients near fp32's smallest and largest keep all their bits: products are exact,
    and a sum loses a step per term at most (and half of fp32's smallest, where it is that small)."""
    r = rng(rows + inp)
    x = (r.standard_normal((rows, inp)) * 2.0 ** xs).astype(np.float32)
    dy = (np.clip(r.standard_normal((rows, out)), -4, 4) * 2.0 ** ds).astype(np.float32)
    got, db = wgrad(hip, x, dy, inp, -(-inp // 32), out, out, np.zeros((inp, out), np.float32), np.zeros(out, np.float32), 0)
    v, d = q8_ref.kept(x).astype(np.float64), dy.astype(np.float64)
    tol = 2 * F32 * (rows + 4) * (np.abs(v).T @ np.abs(d)) + (rows + 4) * 2.0 ** -149
    assert (np.abs(got - v.T @ d) <= tol).all()
    assert (np.abs(db - d.sum(0)) <= 2 * F32 * (rows + 4) * np.abs(d).sum(0) + 2.0 ** -149).all()


@pytest.mark.parametrize("rows,inp,out,acc", [(8, 64, 64, 0), (16, 300, 40, 1), (8, 2048, 2048, 0), (4096, 48, 52, 1)])
def test_linear_wgrad_columns_of_every_size(hip, rows, inp, out, acc):
    """Columns of dY from 2^-122 to 2^116 beside each other in one tile."""
    r = rng(rows + out)
    x = r.standard_normal((rows, inp)).astype(np.float32)
    size = r.choice(np.array([-122, -60, 0, 60, 116]), out)
    dy = (np.clip(r.standard_normal((rows, out)), -4, 4) * np.exp2(size)).astype(np.float32)
    old = (r.standard_normal((inp, out)) * np.exp2(size)).astype(np.float32)
    got, _ = wgrad(hip, x, dy, inp, -(-inp // 32), out, out, old, np.zeros(out, np.float32), acc)
    v, d = q8_ref.kept(x).astype(np.float64), dy.astype(np.float64)
    ref = v.T @ d + (old.astype(np.float64) if acc else 0)
    tol = 2 * F32 * ((rows + 4) * (np.abs(v).T @ np.abs(d)) + 2 * np.abs(old)) + (rows + 4) * 2.0 ** -149
    assert (np.abs(got - ref) <= tol).all()


OTHERS = {  # the function and its derivative
    "tanh": (np.tanh, lambda x: 1 - np.tanh(x) ** 2),
    "sigmoid": (lambda x: 1 / (1 + np.exp(-x)), lambda x: 1 / (2 + np.exp(x) + np.exp(-x))),
    "leaky_relu": (lambda x: np.where(x < 0, 0.01 * x, x), lambda x: np.where(x < 0, 0.01, 1.0)),
}


@pytest.mark.parametrize("kind", OTHERS)
@pytest.mark.parametrize("rows,cols,pad,acc", [(1, 1, 0, 0), (33, 70, 2, 1), (20, 330, 0, 0)])
def test_other_activations(hip, kind, rows, cols, pad, acc):
    """tanh, sigmoid and leaky ReLU: each by its formula, and the elementwise calls' bits."""
    r = rng(cols + 1)
    f, df = OTHERS[kind]
    x = (r.standard_normal((rows, cols)) * 3).astype(np.float32)
    dy, old = (r.standard_normal((rows, cols)).astype(np.float32) for _ in range(2))
    ld, ng = cols + pad, -(-cols // 32)
    B = hip.Buffer
    gx, gy = B.from_array(padded(x, ld, 7.0)), B.from_array(np.full((rows, ld), 5, np.float32))
    gq, ge = B.empty((rows, ld), np.int8), B.empty((rows, ng), np.uint8)
    hip.call("mle_q8_act_fwd", None, hip.ACT[kind], rows, cols, gx.ptr, ld, gy.ptr, ld, gq.ptr, ld, ge.ptr, ng)
    q, e = q8_ref.quantize(x)
    assert np.array_equal(gq.numpy()[:, :cols], q) and np.array_equal(ge.numpy(), e)
    y = gy.numpy()
    # an exponential or a tanh of a few steps, a division and two sums, of values up to 1 or |x|
    assert (np.abs(y[:, :cols] - f(x.astype(np.float64))) <= 16 * F32 * (np.abs(x) + 1)).all() and (y[:, cols:] == 5).all()
    fx, fy = B.from_array(x), B.empty((rows, cols))
    hip.call("mle_act_fwd", None, hip.ACT[kind], fx.ptr, fy.ptr, rows * cols)
    assert np.array_equal(fy.numpy(), y[:, :cols])
    gdy, gdx = B.from_array(padded(dy, ld, 7.0)), B.from_array(padded(old, ld, 3.0))
    hip.call("mle_q8_act_bwd", None, hip.ACT[kind], rows, cols, gq.ptr, ld, ge.ptr, ng, gdy.ptr, ld, gdx.ptr, ld, acc)
    dx, v = gdx.numpy(), q8_ref.values(q, e).astype(np.float64)
    ref = df(v) * dy + (old if acc else 0)
    # the same operations again, of a derivative of at most 1
    assert (np.abs(dx[:, :cols] - ref) <= F32 * (16 * np.abs(dy) + 2 * np.abs(old))).all() and (dx[:, cols:] == 3).all()
    fv, fdy, fdx = B.from_array(v.astype(np.float32)), B.from_array(dy), B.from_array(old)
    hip.call("mle_act_bwd", None, hip.ACT[kind], fv.ptr, fdy.ptr, fdx.ptr, rows * cols, acc)
    assert np.array_equal(fdx.numpy(), dx[:, :cols])


@pytest.mark.parametrize("rows,inp,out", [(100, 96, 40), (8, 2048, 2048), (3000, 48, 52), (20, 3, 70)])
@pytest.mark.parametrize("bad", [0x7F800000, 0xFF800000, 0x7FC00000, 0x7F800001])
def test_linear_wgrad_not_finite_gradients_stay_in_their_column(hip, rows, inp, out, bad):
    """An infinity or a NaN (also one whose payload is in the last bits only) in dY: its
    column of dW is NaN, the others are as they were."""
    r = rng(rows)
    x, dy = r.standard_normal((rows, inp)).astype(np.float32), r.standard_normal((rows, out)).astype(np.float32)
    args = (inp, -(-inp // 32), out, out, np.zeros((inp, out), np.float32), np.zeros(out, np.float32), 0)
    want, want_db = wgrad(hip, x, dy, *args)
    dy.view(np.uint32)[rows // 2, 17] = bad
    got, db = wgrad(hip, x, dy, *args)
    assert np.isnan(got[:, 17]).all() and not np.isfinite(db[17])
    assert np.array_equal(np.delete(got, 17, 1), np.delete(want, 17, 1)) and np.array_equal(np.delete(db, 17), np.delete(want_db, 17))
