"""The vocabulary's two ends in the engine: Embedding::forward with a scale and
Linear::cross_entropy, around one feed-forward, against 64 bits and against the
graph that keeps the logits."""
import math

import numpy as np
import pytest

from conftest import rng
from ml_engine_amd.models import STEP_ALL, STEP_BACKWARD, STEP_FORWARD, STEP_ZERO, Model

pytestmark = pytest.mark.gpu
GRADS = STEP_ZERO | STEP_FORWARD | STEP_BACKWARD


def data(B, S, D, F, V, max_clen, seed=0):
    r = rng(seed)
    u = lambda *s, b: r.uniform(-b, b, s).astype(np.float32)  # noqa: E731
    params = [u(V, D, b=0.2), u(D, F, b=math.sqrt(3 / D)), u(F, b=0.1), u(F, D, b=math.sqrt(3 / F)), u(D, b=0.1),
              u(D, V, b=math.sqrt(3 / D)), u(V, b=0.1)]
    ids, tgt = (r.integers(0, V, (B, max_clen)).astype(np.int32) for _ in range(2))
    ids[0, S // 2:] = -1
    return params, ids, tgt


def model(dims, whole, params, ids, tgt, **kw):
    B, S, D, F, V, mx = dims
    m = Model("language", (B, S, D, F, V, whole, mx), **kw)
    for i, p in enumerate(params):
        m.set(i, p)
    m.input(0, ids)
    m.input(1, tgt)
    return m


def exact(dims, params, ids, tgt):
    """Loss and gradients in 64 bits; positions whose target is outside the vocabulary take no part."""
    B, S, D, F, V, _ = dims
    E, W1, b1, W2, b2, W, b = (p.astype(np.float64) for p in params)
    k, t = ids[:, :S].reshape(-1), tgt[:, :S].reshape(-1)
    ok, tk = k >= 0, (t >= 0) & (t < V)
    s = float(np.float32(math.sqrt(D)))
    x = np.where(ok[:, None], E[np.maximum(k, 0)], 0) * s
    h = x @ W1 + b1
    c = math.sqrt(2 / math.pi)
    th = np.tanh(c * (h + 0.044715 * h ** 3))
    a = 0.5 * h * (1 + th)
    y = x + a @ W2 + b2
    l = y @ W + b
    l -= l.max(1, keepdims=True)
    p = np.exp(l)
    p /= p.sum(1, keepdims=True)
    at, tt = np.arange(B * S), np.where(tk, t, 0)
    loss = -(np.log(p[at, tt]) * tk).sum() / (B * S * V)
    g = p.copy()
    g[at, tt] -= 1
    g *= tk[:, None] / B
    dy = g @ W.T
    da = dy @ W2.T
    dh = da * (0.5 * (1 + th) + 0.5 * h * (1 - th ** 2) * c * (1 + 0.134145 * h ** 2))
    dx = dy + dh @ W1.T
    dE = np.zeros_like(E)
    np.add.at(dE, k[ok], dx[ok] * s)
    return loss, [dE, x.T @ dh, dh.sum(0), a.T @ dy, dy.sum(0), y.T @ g, g.sum(0)]


# one of few rows (pieces of stored logits), one of many (fp16 planes), one with a
# table above the indexed lookup's limit
SHAPES = [(2, 20, 32, 48, 101, 20), (4, 100, 64, 96, 8000, 104), (3, 130, 48, 32, 20000, 130)]


@pytest.mark.parametrize("dims", SHAPES)
@pytest.mark.parametrize("lazy", [True, False])
def test_against_64_bits(dims, lazy):
    B, S, D, F, V, mx = dims
    params, ids, tgt = data(*dims)
    tgt[-1, S - 3:S] = -2 ** 31
    m = model(dims, 1, params, ids, tgt, lazy_zero=lazy)
    loss, grads = exact(dims, params, ids, tgt)
    for _ in range(2):  # the second step's gradients replace the first's
        m.step(1e-3, GRADS)
        m.sync()
        assert abs(m.loss - loss) <= 1e-5 * abs(loss)
        for i, g in enumerate(grads):
            # chains of fp32 products: some 1e-6 of a tensor's largest gradient
            assert np.abs(m.get(i, 1).reshape(g.shape) - g).max() <= 1e-5 * np.abs(g).max(), m.names[i]
    m.close()


@pytest.mark.parametrize("dims", SHAPES[:2])
def test_as_with_logits(dims):
    """The same training as through the Linear and SoftMaxCrossEntropy."""
    params, ids, tgt = data(*dims, seed=1)
    runs = []
    for whole in (1, 0):
        m = model(dims, whole, params, ids, tgt)
        losses = []
        for _ in range(4):
            m.step(1e-3, STEP_ALL)
            m.sync()
            losses.append(m.loss)
        runs.append((losses, [m.get(i) for i in range(len(params))]))
        m.close()
    assert np.allclose(runs[0][0], runs[1][0], rtol=1e-4)
    for p, q, start in zip(runs[0][1], runs[1][1], params):
        # four AdamW steps move a weight by 4e-3; where a gradient is all noise its
        # sign may differ, so compare the bulk
        assert np.mean(np.abs(p - q) > 2e-4) <= 0.02 and not np.array_equal(p, start.reshape(-1))


@pytest.mark.parametrize("dims", SHAPES)
def test_replayed(dims):
    """The recorded pass, replayed between eager work, trains as the eager one does."""
    params, ids, tgt = data(*dims, seed=2)
    a, b = (model(dims, 1, params, ids, tgt) for _ in range(2))
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


@pytest.mark.parametrize("kind", ["language", "block"])
def test_sgd_step_of_the_table(kind):
    """Embedding::UpdateSGD after a scaled lookup (and after a plain one) steps along the
    gradient that the backward forms: the scale is part of it.  Every id occurs once,
    so that both are one token's row, whatever the order of sums."""
    B, S, D, V = 2, 16, 48 if kind == "language" else 64, 97
    r = rng(5)
    if kind == "language":
        params, _, tgt = data(B, S, D, 32, V, S, seed=3)
        m = Model("language", (B, S, D, 32, V, 1, S))
    else:
        m = Model("block", (B, S, D, 2, 32, V))
        params, tgt = [], r.integers(0, V, (B, S)).astype(np.int32)
    for i, p in enumerate(params):
        m.set(i, p)
    m.input(0, r.permutation(V)[: B * S].astype(np.int32).reshape(B, S))
    m.input(1, tgt)
    m.step(0.0, GRADS)
    table, grad, lr = m.get(0).astype(np.float64), m.get(0, 1).astype(np.float64), 0.5
    m.embed_sgd(lr)
    m.sync()
    assert np.count_nonzero(grad) > B * S * D // 2
    # four roundings of the step (the gradient's, the scale's, the rate's, the product's)
    # and one of the sum, each half a step of fp32 at most
    tol = 2.0 ** -24 * (4 * lr * np.abs(grad) + np.abs(table) + lr * np.abs(grad))
    assert (np.abs(m.get(0) - (table - lr * grad)) <= tol).all()
    m.close()
