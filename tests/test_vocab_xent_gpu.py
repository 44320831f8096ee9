"""The vocabulary's cross entropy without stored logits, against 64 bits."""
import numpy as np
import pytest

from conftest import rng

pytestmark = pytest.mark.gpu
STEP = 2.0 ** -23  # a step of fp32: a sum that is truncated loses at most one per term


class Case:
    """Inputs on the device, strided, with what lies past the rows filled."""

    def __init__(self, hip, rows, d, vocab, bias=True, ignored=0.2, pad=0, clen=None, max_clen=None, seed=0, scale=1.0):
        r = rng(seed + rows + d + vocab)
        self.hip, self.rows, self.d, self.vocab = hip, rows, d, vocab
        self.clen = clen or rows
        self.max_clen = max_clen or self.clen
        self.x = (scale * r.standard_normal((rows, d))).astype(np.float32)
        self.w = (r.uniform(-1, 1, (d, vocab)) * np.sqrt(3.0 / d)).astype(np.float32)
        self.b = r.uniform(-1, 1, vocab).astype(np.float32) if bias else None
        self.keys = r.integers(0, vocab, rows).astype(np.int32)
        self.keys[r.random(rows) < ignored] = r.choice(np.array([-1, -2 ** 31, vocab, 2 ** 31 - 1]))
        self.pad = pad
        self.scale = 1.0 / max(1, int(self.valid().sum()))

    def valid(self):
        return (self.keys >= 0) & (self.keys < self.vocab)

    def put(self):
        wide = lambda a, n: np.concatenate([a, np.full((a.shape[0], n), np.nan, np.float32)], axis=1)  # noqa: E731
        full = np.full((self.rows // self.clen, self.max_clen), 1, np.int32)
        full[:, : self.clen] = self.keys.reshape(-1, self.clen)
        B = self.hip.Buffer
        self.gx, self.gw = B.from_array(wide(self.x, self.pad)), B.from_array(wide(self.w, self.pad))
        self.gb = B.from_array(self.b) if self.b is not None else None
        self.gk = B.from_array(full)
        self.ws = B(self.hip.lib().mle_vocab_xent_ws_bytes(self.rows, self.d, self.vocab))
        self.lse, self.row_loss, self.loss = B.empty(self.rows), B.empty(self.rows), B.empty(1)

    def shape(self):
        return (self.rows, self.d, self.vocab, self.gx.ptr, self.d + self.pad, self.gw.ptr, self.vocab + self.pad,
                self.gb.ptr if self.gb else None, self.gk.ptr, self.clen, self.max_clen)

    def forward(self, stream=None):
        self.hip.call("mle_vocab_xent_fwd", stream, *self.shape(), self.scale, self.lse.ptr, self.row_loss.ptr, self.loss.ptr,
                      self.ws.ptr, self.ws.nbytes)
        return self.lse.numpy(), self.row_loss.numpy(), float(self.loss.numpy()[0])

    def backward(self, acc=0, upstream=None, want=("dx", "dw", "db"), old=0.0, stream=None):
        B = self.hip.Buffer
        full = lambda *s: B.from_array(np.full(s, old, np.float32))  # noqa: E731
        self.gdx, self.gdw, self.gdb = full(self.rows, self.d + self.pad), full(self.d, self.vocab + self.pad), full(self.vocab)
        up = B.from_array(np.array([upstream], np.float32)) if upstream is not None else None
        self.hip.call("mle_vocab_xent_bwd", stream, *self.shape(), self.lse.ptr, up.ptr if up else None, self.scale,
                      self.gdx.ptr if "dx" in want else None, self.d + self.pad, acc, self.gdw.ptr if "dw" in want else None,
                      self.vocab + self.pad, self.gdb.ptr if "db" in want else None, acc, self.ws.ptr, self.ws.nbytes)
        dx, dw, db = self.gdx.numpy(), self.gdw.numpy(), self.gdb.numpy()
        assert (dx[:, self.d:] == np.float32(old)).all() and (dw[:, self.vocab:] == np.float32(old)).all()
        return dx[:, : self.d], dw[:, : self.vocab], db

    def exact(self, upstream=1.0):
        """Values in 64 bits, and how far fp32 sums may be from them."""
        x, w = self.x.astype(np.float64), self.w.astype(np.float64)
        b = self.b.astype(np.float64) if self.b is not None else np.zeros(self.vocab)
        ok, at = self.valid(), np.arange(self.rows)
        l = x @ w + b
        top = l.max(1, keepdims=True)
        e = np.exp(l - top)
        lse = (top + np.log(e.sum(1, keepdims=True)))[:, 0]
        k = np.where(ok, self.keys, 0)
        row_loss = np.where(ok, lse - l[at, k], 0)
        p = np.exp(l - lse[:, None])
        # a logit: a step per product and for the bias; lse: the largest logit's
        # error, the sum's relative one, and the final operations'
        dl = STEP * ((self.d + 4) * (np.abs(x) @ np.abs(w)) + 2 * np.abs(b))
        dlse = (p * dl).sum(1) + STEP * (8 + np.log2(self.vocab) + 2 * np.abs(lse) + 2 * np.abs(top[:, 0]))
        # (a probability below 2^-126 is no normal number: it may come out as 0)
        dp = p * (dl + dlse[:, None] + STEP * (8 + np.abs(l) + np.abs(lse)[:, None])) + 2.0 ** -126
        p[at, k] -= ok
        dp[at, k] += STEP
        g = ok[:, None] * self.scale * upstream
        p, dp = p * g, (dp + 4 * STEP * np.abs(p)) * np.abs(g)
        x0 = np.where(ok[:, None], x, 0)
        out = dict(lse=lse, row_loss=row_loss, loss=row_loss.sum() * self.scale, dx=p @ w.T, dw=x0.T @ p, db=p.sum(0))
        tol = dict(lse=dlse, row_loss=ok * (dlse + dl[at, k] + 2 * STEP * np.abs(row_loss)),
                   dx=dp @ np.abs(w.T) + (self.vocab + 4) * STEP * (np.abs(p) @ np.abs(w.T)),
                   dw=np.abs(x0.T) @ dp + (self.rows + 4) * STEP * (np.abs(x0.T) @ np.abs(p)),
                   db=dp.sum(0) + (self.rows + 4) * STEP * np.abs(p).sum(0))
        tol["loss"] = self.scale * tol["row_loss"].sum() + 4 * STEP * abs(out["loss"])
        return out, tol


def close(got, ref, tol, what):
    err = np.abs(np.asarray(got, np.float64) - ref)
    assert (err <= tol).all(), f"{what}: {np.max(err / np.maximum(tol, 1e-300)):.3g} times the bound"


# few logits (stored in pieces; up to 64 rows and many columns with a kernel of their own
# for dW), then products of fp16 planes: rows and vocabularies on both sides of whole
# tiles, features on both sides of whole stages, several chunks of rows and pieces of
# the vocabulary
SHAPES = [(1, 1, 1), (1, 8, 100), (3, 33, 70), (64, 64, 1000), (64, 256, 4096), (100, 31, 257), (130, 96, 129), (300, 330, 1007),
          (2048, 64, 300), (5, 512, 20011),
          (128, 33, 24001), (300, 330, 10007), (513, 64, 6400), (1030, 65, 3001), (4001, 31, 777), (2048, 128, 1500),
          (33001, 16, 1100), (17, 40, 2051), (2100, 16, 1200), (193, 33, 24001), (200, 3, 24001),
          (250, 1, 25000), (64, 3, 530000), (33, 300, 22001), (64, 130, 33001)]


@pytest.mark.parametrize("rows,d,vocab", SHAPES)
@pytest.mark.parametrize("bias,pad,acc", [(True, 0, 0), (False, 3, 1), (True, 4, 1)])
def test_against_64_bits(hip, rows, d, vocab, bias, pad, acc):
    c = Case(hip, rows, d, vocab, bias, pad=pad)
    c.put()
    ref, tol = c.exact(upstream=0.75)
    lse, row_loss, loss = c.forward()
    close(lse, ref["lse"], tol["lse"], "lse")
    close(row_loss, ref["row_loss"], tol["row_loss"], "row_loss")
    close(loss, ref["loss"], tol["loss"], "loss")
    old = 0.25
    dx, dw, db = c.backward(acc=acc, upstream=0.75, old=old)
    for name, got in (("dx", dx), ("dw", dw), ("db", db)):
        base = old if acc else 0.0
        close(got, ref[name] + base, tol[name] + 2 * STEP * (base + np.abs(ref[name])), name)
    assert acc or (dx[~c.valid()] == 0).all()


@pytest.mark.parametrize("clen,max_clen", [(20, 20), (20, 27)])
def test_padded_sequences(hip, clen, max_clen):
    c = Case(hip, 120, 48, 333, clen=clen, max_clen=max_clen)
    c.put()
    ref, tol = c.exact()
    _, row_loss, _ = c.forward()
    close(row_loss, ref["row_loss"], tol["row_loss"], "row_loss")
    close(c.backward()[1], ref["dw"], tol["dw"], "dw")


@pytest.mark.parametrize("rows,vocab", [(40, 500), (1000, 3100), (48, 66000)])
def test_what_rows_outside_hold_stays_there(hip, rows, vocab):
    """NaN, infinity and huge values in rows that take no part: the loss, dW, db and the other rows' dX as without them."""
    c = Case(hip, rows, 64, vocab, ignored=0.3)
    bad = np.flatnonzero(~c.valid())
    c.x[bad] = 0
    c.put()
    ref, tol = c.exact()
    c.x[bad[::3]] = np.nan
    c.x[bad[1::3], 3] = -np.inf
    c.x[bad[2::3]] = 3e38
    c.put()
    _, row_loss, loss = c.forward()
    dx, dw, db = c.backward()
    # (not the same bits: a tile of products that meets a NaN is multiplied
    # again in fp32, whose sums round elsewhere within the same bounds)
    for name, got in (("row_loss", row_loss), ("loss", loss), ("dx", dx), ("dw", dw), ("db", db)):
        close(got, ref[name], tol[name], name)


@pytest.mark.parametrize("rows,vocab", [(70, 200), (1001, 3003)])
def test_no_row_takes_part(hip, rows, vocab):
    c = Case(hip, rows, 32, vocab, ignored=1.1)
    c.put()
    _, row_loss, loss = c.forward()
    dx, dw, db = c.backward()
    assert loss == 0 and not row_loss.any() and not dx.any() and not dw.any() and not db.any()


@pytest.mark.parametrize("rows,vocab", [(33, 400), (1000, 4600), (48, 66000)])
def test_masked_entries(hip, rows, vocab):
    """A bias of -infinity: as if the entry were not in the vocabulary."""
    c = Case(hip, rows, 64, vocab)
    out = np.arange(0, vocab, 3)
    c.keys[np.isin(c.keys, out) & c.valid()] -= 1
    c.keys[c.keys == -1] = 1
    keep = np.setdiff1d(np.arange(vocab), out)
    c.b[out] = -np.inf
    c.w[:, out[::2]] *= 1e30  # what no entry holds
    c.put()
    lse, row_loss, _ = c.forward()
    dx, dw, db = c.backward()
    small = Case(hip, rows, 64, keep.size)
    small.x, small.w, small.b, small.scale = c.x, np.ascontiguousarray(c.w[:, keep]), c.b[keep], c.scale
    small.keys = np.where(c.valid(), np.searchsorted(keep, np.where(c.valid(), c.keys, keep[0])), -1).astype(np.int32)
    ref, tol = small.exact()
    close(lse, ref["lse"], tol["lse"], "lse")
    close(row_loss, ref["row_loss"], tol["row_loss"], "row_loss")
    close(dx, ref["dx"], tol["dx"], "dx")
    close(dw[:, keep], ref["dw"], tol["dw"], "dw")
    assert not dw[:, out].any() and not db[out].any()


@pytest.mark.parametrize("rows,vocab", [(40, 300), (1030, 3000), (48, 66000)])
@pytest.mark.parametrize("size", [1.0, 60.0, 2.0 ** -30])
def test_rows_outside_have_their_log_sum(hip, rows, vocab, size):
    """Ordinary values there, other than the rest's: lse is theirs.  Some features are
    zero in every row that takes part."""
    c = Case(hip, rows, 64, vocab, ignored=0.4)
    c.x[~c.valid()] *= np.float32(size)
    c.x[np.ix_(c.valid(), np.arange(5))] = 0
    c.put()
    ref, tol = c.exact()
    close(c.forward()[0], ref["lse"], tol["lse"], "lse")
    dx, dw, db = c.backward()
    for name, got in (("dx", dx), ("dw", dw), ("db", db)):
        close(got, ref[name], tol[name], name)


@pytest.mark.parametrize("rows,vocab", [(30, 200), (1000, 3100), (48, 66000)])
def test_unaligned_buffers(hip, rows, vocab):
    """Every float buffer begins 4 bytes past an aligned address."""
    c = Case(hip, rows, 36, vocab)
    c.put()
    ref, tol = c.exact()
    B = hip.Buffer
    off = lambda a: B.from_array(np.concatenate([np.zeros(1, np.float32), a.reshape(-1).astype(np.float32)]))  # noqa: E731
    gx, gw, gb = off(c.x), off(c.w), off(c.b)
    out = {k: off(np.zeros(n)) for k, n in (("lse", rows), ("row_loss", rows), ("loss", 1), ("dx", rows * 36),
                                            ("dw", 36 * vocab), ("db", vocab))}
    p = {k: v.ptr + 4 for k, v in out.items()}
    shape = (rows, 36, vocab, gx.ptr + 4, 36, gw.ptr + 4, vocab, gb.ptr + 4, c.gk.ptr, rows, rows)
    hip.call("mle_vocab_xent_fwd", None, *shape, c.scale, p["lse"], p["row_loss"], p["loss"], c.ws.ptr, c.ws.nbytes)
    hip.call("mle_vocab_xent_bwd", None, *shape, p["lse"], None, c.scale, p["dx"], 36, 0, p["dw"], vocab, p["db"], 0, c.ws.ptr,
             c.ws.nbytes)
    for k, v in out.items():
        close(v.numpy()[1:], np.asarray(ref[k]).reshape(-1), np.asarray(tol[k]).reshape(-1), k)


@pytest.mark.parametrize("rows,vocab", [(20, 300), (1030, 3000), (48, 66000)])
def test_not_finite_rows(hip, rows, vocab):
    """A NaN in a row that takes part: its lse and the loss are NaN, other rows' values stay."""
    c = Case(hip, rows, 64, vocab, ignored=0.0)
    c.put()
    ref, tol = c.exact()
    c.x[7, 5] = np.nan
    c.put()
    lse, row_loss, loss = c.forward()
    assert np.isnan(lse[7]) and np.isnan(row_loss[7]) and np.isnan(loss)
    close(np.delete(lse, 7), np.delete(ref["lse"], 7), np.delete(tol["lse"], 7), "lse")
    dx, dw, _ = c.backward()
    assert np.isnan(dx[7]).all() and np.isfinite(np.delete(dx, 7, 0)).all() and np.isnan(dw).all()


@pytest.mark.parametrize("rows,vocab", [(50, 700), (1100, 2900), (48, 66000)])
def test_parts_of_the_gradient(hip, rows, vocab):
    """dX alone, dW alone, dW without db, and no row losses."""
    c = Case(hip, rows, 96, vocab)
    c.put()
    ref, tol = c.exact()
    c.forward()
    for want in (("dx",), ("dw",), ("dw", "db"), ("dx", "dw"), ("dx", "dw", "db")):
        got = dict(zip(("dx", "dw", "db"), c.backward(want=want, old=9.0)))
        for name, v in got.items():
            if name in want:
                close(v, ref[name], tol[name], name)
            else:
                assert (v == 9.0).all(), name
    lse, loss = c.lse.numpy(), c.loss.numpy()
    c.hip.call("mle_vocab_xent_fwd", None, *c.shape(), c.scale, c.lse.ptr, None, c.loss.ptr, c.ws.ptr, c.ws.nbytes)
    assert np.array_equal(c.lse.numpy(), lse) and np.array_equal(c.loss.numpy(), loss)


@pytest.mark.parametrize("scale", [2.0 ** -40, 60.0])
@pytest.mark.parametrize("rows,vocab", [(48, 600), (1030, 3000), (48, 66000)])
def test_small_and_confident_rows(hip, rows, vocab, scale):
    """Rows of tiny values (a flat softmax), and logits up to some hundreds."""
    c = Case(hip, rows, 64, vocab, scale=scale)
    c.put()
    ref, tol = c.exact()
    lse, row_loss, _ = c.forward()
    close(lse, ref["lse"], tol["lse"], "lse")
    close(row_loss, ref["row_loss"], tol["row_loss"], "row_loss")
    dx, dw, db = c.backward()
    close(dx, ref["dx"], tol["dx"], "dx")
    close(dw, ref["dw"], tol["dw"], "dw")
    close(db, ref["db"], tol["db"], "db")


@pytest.mark.parametrize("rows,vocab", [(64, 500), (1024, 3000), (48, 66000)])
def test_values_of_very_different_size(hip, rows, vocab):
    """Columns of X and rows of W from 2^-30 to 2^30 of each other."""
    c = Case(hip, rows, 64, vocab)
    f = np.exp2(rng(1).integers(-30, 31, 64)).astype(np.float32)
    c.x = (c.x * f).astype(np.float32)
    c.w = (c.w / f[:, None]).astype(np.float32)
    c.put()
    ref, tol = c.exact()
    close(c.forward()[0], ref["lse"], tol["lse"], "lse")
    dx, dw, _ = c.backward()
    close(dx, ref["dx"], tol["dx"], "dx")
    close(dw, ref["dw"], tol["dw"], "dw")


@pytest.mark.parametrize("rows,d,vocab", [(64, 256, 4096), (1024, 256, 4000), (2048, 512, 2000)])
def test_two_norm(hip, rows, d, vocab):
    """The error of a typical case in the 2-norm: that of fp32 products, well
    under the worst-case bounds above (24 bits each, random in sign)."""
    c = Case(hip, rows, d, vocab, ignored=0.0)
    c.put()
    ref, _ = c.exact()
    lse, _, _ = c.forward()
    dx, dw, db = c.backward()
    for got, want in ((lse, ref["lse"]), (dx, ref["dx"]), (dw, ref["dw"]), (db, ref["db"])):
        assert np.linalg.norm(got - want) <= 2e-6 * np.linalg.norm(want)


@pytest.mark.parametrize("rows,vocab", [(60, 900), (1000, 3100), (48, 66000)])
def test_repeats(hip, rows, vocab):
    c = Case(hip, rows, 80, vocab)
    c.put()
    a = (*c.forward(), *c.backward())
    b = (*c.forward(), *c.backward())
    for u, v in zip(a, b):
        assert np.array_equal(u, v)


def test_gradient_against_differences(hip):
    c = Case(hip, 6, 10, 30, ignored=0.3)
    c.put()
    c.forward()
    dx, dw, db = c.backward()

    def f(x, w, b):
        l = x @ w + b
        m = l.max(1)
        z = m + np.log(np.exp(l - m[:, None]).sum(1))
        ok = c.valid()
        return float((z - l[np.arange(6), np.where(ok, c.keys, 0)])[ok].sum() * c.scale)

    args, h = [a.astype(np.float64) for a in (c.x, c.w, c.b)], 1e-5
    for n, grad in enumerate((dx, dw, db)):
        for i in np.ndindex(*args[n].shape):
            d = [a.copy() for a in args]
            d[n][i] += h
            up = f(*d)
            d[n][i] -= 2 * h
            # the difference's own error is about h^2 and 1e-16 / h
            assert abs((up - f(*d)) / (2 * h) - grad[i]) <= 1e-6


def test_no_rows(hip):
    w, loss = hip.Buffer.from_array(np.ones((8, 20), np.float32)), hip.Buffer.from_array(np.ones(1, np.float32))
    dw, db = hip.Buffer.from_array(np.ones((8, 20), np.float32)), hip.Buffer.from_array(np.ones(20, np.float32))
    shape = (0, 8, 20, None, 8, w.ptr, 20, None, None, 1, 1)
    hip.call("mle_vocab_xent_fwd", None, *shape, 1.0, None, None, loss.ptr, None, 0)
    assert loss.numpy()[0] == 0
    hip.call("mle_vocab_xent_bwd", None, *shape, None, None, 1.0, None, 8, 0, dw.ptr, 20, db.ptr, 1, None, 0)
    assert (dw.numpy() == 1).all() and (db.numpy() == 1).all()
    hip.call("mle_vocab_xent_bwd", None, *shape, None, None, 1.0, None, 8, 0, dw.ptr, 20, db.ptr, 0, None, 0)
    assert not dw.numpy().any() and not db.numpy().any()


@pytest.mark.parametrize("rows,d,vocab", [(8, 16, 66000), (48, 64, 66000), (8, 64, 900), (256, 16, 13000)])
@pytest.mark.parametrize("size,upstream", [(0, -104), (-120, 40), (108, 0), (0, 90)])
def test_gradients_near_the_smallest_and_the_largest(hip, rows, d, vocab, size, upstream):
    """X of 2^size against W of 2^-size, and a scaled loss: P or X near fp32's smallest numbers,
    or X near its largest, on a softmax that is the same."""
    c = Case(hip, rows, d, vocab, ignored=0.2)
    c.x = (c.x * 2.0 ** size).astype(np.float32)
    c.w = (c.w * 2.0 ** min(-size, 80)).astype(np.float32)
    if size == 108:
        c.w = (c.w * 2.0 ** -8).astype(np.float32)
    c.put()
    ref, tol = c.exact(upstream=2.0 ** upstream)
    c.forward()
    dx, dw, db = c.backward(upstream=2.0 ** upstream)
    # (what is below 2^-126 holds multiples of 2^-149: half a one for each P and each sum)
    x = np.abs(np.where(c.valid()[:, None], c.x, 0).astype(np.float64))
    w = np.abs(c.w.astype(np.float64))
    small = 2.0 ** -149
    close(dw, ref["dw"], tol["dw"] + small * (x.sum(0)[:, None] + rows + 4), "dw")
    close(dx, ref["dx"], tol["dx"] + small * (w.sum(1) + vocab + 4), "dx")
    close(db, ref["db"], tol["db"] + small * (2 * rows + 4), "db")


# few logits, with the library's product and with dW's own kernel; planes of 128 and
# of several hundred rows
@pytest.mark.parametrize("rows,vocab", [(60, 900), (48, 66000), (256, 13000), (700, 6000)])
@pytest.mark.parametrize("gap", [7, 12, 17])
def test_small_probabilities_beside_targets(hip, rows, vocab, gap):
    """Columns that are some rows' targets and hardly likely in the others, which alone have
    certain features: those entries of dW are sums of small P and as exact as large ones,
    down to 2^-50 of the column's largest P."""
    r = rng(rows + gap)
    d, hot = 8, 16
    c = Case(hip, rows, d, vocab, bias=False, ignored=0.0)
    target = np.arange(rows) % 64 < hot  # rows with a hot column as their id, in every 64
    c.keys = np.where(target, np.arange(rows) % 64, r.integers(hot, vocab, rows)).astype(np.int32)
    c.x = r.standard_normal((rows, d)).astype(np.float32)
    c.x[target, 1:] = 0
    c.x[:, 0] = 1
    c.w = np.zeros((d, vocab), np.float32)  # logits: -gap in hot columns, 0 in the others
    c.w[0, :hot] = -gap
    c.put()
    c.forward()
    _, dw, _ = c.backward()
    lse = np.log(hot * np.exp(-gap) + (vocab - hot))
    p = np.exp(-gap - lse) * c.scale
    x = c.x[~target, 1:].astype(np.float64)
    # the logits are whole numbers; the sum of their exponentials, its logarithm, the
    # difference and its exponential, the scale, then the products' sum
    rel = STEP * (16 + np.log2(vocab) + 2 * gap + 2 * lse + rows + 4)
    tol = np.abs(x).sum(0) * (p * rel + 2.0 ** -50 * c.scale)
    close(dw[1:, :hot], np.repeat((x.sum(0) * p)[:, None], hot, 1), tol[:, None], "dw")


@pytest.mark.parametrize("rows,vocab", [(60, 900), (48, 66000), (256, 13000), (700, 6000)])
@pytest.mark.parametrize("ratio", [20, 34])
def test_small_rows_beside_a_large_one(hip, rows, vocab, ratio):
    """A feature that one row has 2^ratio times as large as the others: columns that this row
    gives no probability keep the others' bits, down to 2^-50 of the feature's largest value."""
    r = rng(rows + ratio)
    d, cold = 8, 16
    c = Case(hip, rows, d, vocab, bias=False, ignored=0.0)
    c.keys = r.integers(cold, vocab, rows).astype(np.int32)
    c.x = r.standard_normal((rows, d)).astype(np.float32)
    c.x[:, 0] = 0
    c.x[5, 0] = 1       # this row's logits of the cold columns are -300: their P is zero
    c.x[5, 1:] = 2.0 ** ratio
    c.w = np.zeros((d, vocab), np.float32)
    c.w[0, :cold] = -300
    c.put()
    c.forward()
    _, dw, _ = c.backward()
    others = np.delete(c.x, 5, 0)[:, 1:].astype(np.float64)
    p, lse = c.scale / vocab, np.log(vocab)
    rel = STEP * (16 + np.log2(vocab) + 2 * lse + rows + 4)
    tol = p * (np.abs(others).sum(0) * rel + 2.0 ** (ratio - 50) * rows)
    close(dw[1:, :cold], np.repeat((others.sum(0) * p)[:, None], cold, 1), tol[:, None], "dw")


@pytest.mark.parametrize("rows,vocab", [(33, 400), (5, 20011), (48, 66000), (1000, 4600)])
@pytest.mark.parametrize("big", [3e38, 1e20])
def test_masked_entries_of_any_weights(hip, rows, vocab, big):
    """Entries that the bias takes out, with weights whose products overflow (both signs in a
    sum): as if their weights were zero."""
    c = Case(hip, rows, 64, vocab)
    out = np.arange(0, vocab, 3)
    c.keys[np.isin(c.keys, out) & c.valid()] += 1
    c.b[out] = 0
    c.w[:, out] = 0
    ref_b = c.b.copy()
    c.b[out] = -1e9  # no probability left in 64 bits either
    ref, tol = c.exact()
    c.b = ref_b
    c.b[out] = -np.inf
    c.w[:, out] = (big * rng(vocab).choice(np.array([-1, 1]), (64, out.size))).astype(np.float32)
    c.put()
    lse, row_loss, loss = c.forward()
    dx, dw, db = c.backward()
    keep = np.setdiff1d(np.arange(vocab), out)
    close(lse, ref["lse"], tol["lse"] + STEP * np.abs(ref["lse"]), "lse")
    close(row_loss, ref["row_loss"], tol["row_loss"] + STEP * np.abs(ref["row_loss"]), "row_loss")
    close(dx, ref["dx"], tol["dx"], "dx")
    close(dw[:, keep], ref["dw"][:, keep], tol["dw"][:, keep], "dw")
    assert not dw[:, out].any() and not db[out].any()
