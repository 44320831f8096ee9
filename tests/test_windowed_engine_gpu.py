"""A transformer block in the engine: AffineLayerNorm, WindowSelfAttention (rotary positions, a
window, sinks, shared heads of keys, padded sequences) and a feed-forward between the vocabulary's
two ends, against 64 bits, lazily cleared and fused or not, and replayed."""
import math

import numpy as np
import pytest

from conftest import rng
from ml_engine_amd.models import STEP_ALL, STEP_BACKWARD, STEP_FORWARD, STEP_ZERO, Model

pytestmark = pytest.mark.gpu
GRADS = STEP_ZERO | STEP_FORWARD | STEP_BACKWARD
EPS = float(np.float32(1e-5))


def data(dims, seed=0):
    B, S, D, H, G, hd, F, V, _, _, axes = dims
    r = rng(seed)
    u = lambda *s, b: r.uniform(-b, b, s).astype(np.float32)  # noqa: E731
    lin = lambda n, p: [u(n, p, b=math.sqrt(3 / n)), u(p, b=0.1)]  # noqa: E731
    norm = lambda: [1 + u(D, b=0.5), u(D, b=0.2)]  # noqa: E731
    params = [u(V, D, b=0.2), *norm(), *lin(D, H * hd), *lin(D, G * hd), *lin(D, G * hd), *lin(H * hd, D), *norm(),
              *lin(D, F), *lin(F, D), *norm(), *lin(D, V)]
    ids, tgt = (r.integers(0, V, (B, S)).astype(np.int32) for _ in range(2))
    pos = np.stack([r.permutation(4 * S)[:S] if a else np.arange(S) for a in range(axes) for _ in range(B)])
    lengths = r.integers(1, S + 1, B).astype(np.int32)
    lengths[0] = S
    for b in range(B):
        tgt[b, lengths[b]:] = -1
    return params, (ids, tgt, pos.reshape(axes, B, S).astype(np.int32), lengths)


def model(dims, params, inputs, **kw):
    m = Model("windowed", dims, **kw)
    for i, p in enumerate(params):
        m.set(i, p)
    for i, x in enumerate(inputs):
        m.input(i, x)
    return m


def exact(dims, params, inputs):
    """Loss and gradients in 64 bits."""
    B, S, D, H, G, hd, F, V, window, sinks, axes = dims
    ids, tgt, pos, lengths = inputs
    P = [p.astype(np.float64) for p in params]
    E, w1, c1, Wq, bq, Wk, bk, Wv, bv, Wo, bo, w2, c2, W1, b1, W2, b2, w3, c3, W, bias = P
    s = float(np.float32(math.sqrt(D)))
    x = E[ids.reshape(-1)] * s

    def norm(h, w, c):
        d = h - h.mean(1, keepdims=True)
        r = 1 / np.sqrt((d * d).mean(1, keepdims=True) + EPS)
        return d * r * w + c, (d * r, r, w)

    def norm_back(dy, kept):
        u, r, w = kept
        g = dy * w
        return r * (g - g.mean(1, keepdims=True) - u * (g * u).mean(1, keepdims=True)), (dy * u).sum(0), dy.sum(0)

    n = hd // 2
    sections = [n * (i + 1) // axes - n * i // axes for i in range(axes)]
    axis = np.repeat(np.arange(axes), sections)
    angle = pos.reshape(axes, -1)[axis].T.astype(np.float64) * 10000.0 ** -(np.arange(n) / n)
    co, si = np.cos(angle)[:, None], np.sin(angle)[:, None]

    def turn(t, back=1):
        t = t.reshape(B * S, -1, hd)
        y = t.copy()
        a, b = t[:, :, :n], t[:, :, n:2 * n]
        y[:, :, :n], y[:, :, n:2 * n] = a * co - back * b * si, back * a * si + b * co
        return y

    y1, k1 = norm(x, w1, c1)
    q, k, v = turn(y1 @ Wq + bq), turn(y1 @ Wk + bk), (y1 @ Wv + bv).reshape(B * S, G, hd)
    scale = float(np.float32(1 / np.sqrt(np.float32(hd))))
    i, j = np.arange(S)[:, None], np.arange(S)[None]
    see = (j <= i) & ((i - j < window) | (j < sinks))
    out = np.zeros((B * S, H, hd))
    kept = {}
    for b in range(B):
        L = lengths[b]
        at = slice(b * S, b * S + L)
        for h in range(H):
            e = h * G // H
            z = np.where(see[:L, :L], scale * (q[at, h] @ k[at, e].T), -np.inf)
            p = np.exp(z - z.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            out[at, h] = p @ v[at, e]
            kept[b, h] = p
    h = x + out.reshape(B * S, -1) @ Wo + bo
    y2, k2 = norm(h, w2, c2)
    f = y2 @ W1 + b1
    c = math.sqrt(2 / math.pi)
    th = np.tanh(c * (f + 0.044715 * f ** 3))
    act = 0.5 * f * (1 + th)
    y3, k3 = norm(h + act @ W2 + b2, w3, c3)
    l = y3 @ W + bias
    l -= l.max(1, keepdims=True)
    p = np.exp(l)
    p /= p.sum(1, keepdims=True)
    t = tgt.reshape(-1)
    tk = (t >= 0) & (t < V)
    rows = np.arange(B * S)
    t = np.where(tk, t, 0)
    loss = -(np.log(p[rows, t]) * tk).sum() / (B * S * V)
    g = p.copy()
    g[rows, t] -= 1
    g *= tk[:, None] / B
    dx3, dw3, dc3 = norm_back(g @ W.T, k3)
    df = dx3 @ W2.T * (0.5 * (1 + th) + 0.5 * f * (1 - th ** 2) * c * (1 + 0.134145 * f ** 2))
    dh, dw2, dc2 = norm_back(df @ W1.T, k2)
    dh = dh + dx3
    do = (dh @ Wo.T).reshape(B * S, H, hd)
    dq, dk, dv = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
    for (b, a), pr in kept.items():
        at, e = slice(b * S, b * S + lengths[b]), a * G // H
        dp = do[at, a] @ v[at, e].T
        ds = pr * (dp - (pr * dp).sum(1, keepdims=True))
        dq[at, a] = scale * ds @ k[at, e]
        dk[at, e] += scale * ds.T @ q[at, a]
        dv[at, e] += pr.T @ do[at, a]
    dq, dk, dv = (t.reshape(B * S, -1) for t in (turn(dq, -1), turn(dk, -1), dv))
    dx, dw1, dc1 = norm_back(dq @ Wq.T + dk @ Wk.T + dv @ Wv.T, k1)
    dE = np.zeros_like(E)
    np.add.at(dE, ids.reshape(-1), (dx + dh) * s)
    return loss, [dE, dw1, dc1, y1.T @ dq, dq.sum(0), y1.T @ dk, dk.sum(0), y1.T @ dv, dv.sum(0),
                  out.reshape(B * S, -1).T @ dh, dh.sum(0), dw2, dc2, y2.T @ df, df.sum(0), act.T @ dx3, dx3.sum(0),
                  dw3, dc3, y3.T @ g, g.sum(0)]


# B, S, D, heads, heads of keys, head_dim, F, V, window, sinks, axes
SHAPES = [(2, 20, 32, 4, 2, 8, 48, 101, 7, 2, 1), (3, 130, 64, 4, 4, 16, 96, 300, 50, 3, 2),
          (2, 201, 48, 6, 3, 46, 64, 500, 64, 0, 3), (2, 150, 64, 2, 1, 80, 32, 200, 400, 4, 1)]


@pytest.mark.parametrize("dims", SHAPES)
@pytest.mark.parametrize("kw", [{}, dict(lazy_zero=False), dict(fuse=False)], ids=["", "eager", "unfused"])
def test_against_64_bits(dims, kw):
    params, inputs = data(dims)
    m = model(dims, params, inputs, **kw)
    loss, grads = exact(dims, params, inputs)
    for _ in range(2):  # the second step's gradients replace the first's
        m.step(1e-3, GRADS)
        m.sync()
        assert abs(m.loss - loss) <= 2e-5 * abs(loss)
        for i, g in enumerate(grads):
            # up to 28 passes one after the other, each off by at most some 1.5e-6 of the largest
            # (sums of 200 fp32 products at 2^-24, operands at 2^-22); a key's bias has a
            # gradient that is all noise where nothing turns: of the weight's size, then
            size = max(np.abs(g).max(), np.abs(grads[i - 1]).max() if m.names[i].endswith("Key B1") else 0)
            assert np.abs(m.get(i, 1).reshape(g.shape) - g).max() <= 4.2e-5 * size, m.names[i]
    m.close()


@pytest.mark.parametrize("dims", SHAPES)
def test_replayed(dims):
    """The recorded pass, replayed between eager work, trains as the eager one does."""
    params, inputs = data(dims, seed=2)
    a, b = (model(dims, params, inputs) for _ in range(2))
    for step in range(4):
        a.step(1e-3, STEP_ALL)
        b.step_graph(1e-3, STEP_ALL)
        a.sync()
        b.sync()
        assert a.loss == b.loss, step
        for i in range(len(params)):
            assert np.array_equal(a.get(i, 1), b.get(i, 1)) and np.array_equal(a.get(i), b.get(i)), (step, i)
    a.close()
    b.close()


def test_new_lengths_between_steps():
    """Lengths, positions and ids are read in every pass, the recorded one's among them."""
    dims = SHAPES[1]
    params, first = data(dims, seed=3)
    _, other = data(dims, seed=4)
    m = model(dims, params, first)
    for inputs in (first, other, first):
        for i, x in enumerate(inputs):
            m.input(i, x)
        loss, grads = exact(dims, params, inputs)
        m.step_graph(1e-3, GRADS)
        m.sync()
        assert abs(m.loss - loss) <= 2e-5 * abs(loss)
        for i, g in enumerate(grads):
            assert np.abs(m.get(i, 1).reshape(g.shape) - g).max() <= 4.2e-5 * np.abs(g).max(), m.names[i]
    m.close()


def test_initial_norms_and_checkpoint(tmp_path):
    """Weights start at 1, biases at 0, and a checkpoint brings back what was trained."""
    dims = SHAPES[0]
    params, inputs = data(dims, seed=5)
    m = Model("windowed", dims)
    for i, name in enumerate(m.names):
        if name.startswith("Norm"):
            assert (m.get(i) == (1 if name.endswith("W1") else 0)).all()
    for i, x in enumerate(inputs):
        m.input(i, x)
    for _ in range(2):
        m.step(1e-3, STEP_ALL)
    m.sync()
    m.save(tmp_path / "block.ckpt")
    fresh = Model("windowed", dims, seed=7)
    fresh.load(tmp_path / "block.ckpt")
    for i in range(len(m.names)):
        for which in (0, 2, 3):
            assert np.array_equal(m.get(i, which), fresh.get(i, which)), m.names[i]
    m.close()
    fresh.close()
