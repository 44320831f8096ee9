"""Attention with a sliding window and sinks against 64 bits: forward, backward and
the single-token form, at sizes around tiles, masks, padded batches, strides,
values that are not finite, and under capture."""
import ctypes as C

import numpy as np
import pytest

import wattn_ref as ref
from conftest import rng

pytestmark = pytest.mark.gpu


class Field:
    """A [batch, rows, heads * dim] tensor with a leading dimension and a start of its own on the device."""

    def __init__(self, hip, a, pad=0, shift=0):
        b, n, h, d = a.shape
        self.shape, self.ld, self.shift = a.shape, h * d + pad, shift
        full = np.full((b, n, self.ld), np.float32(7.5))
        full[:, :, :h * d] = a.reshape(b, n, h * d)
        self.buf = hip.Buffer.from_array(np.concatenate([np.full(shift, np.float32(7.5)), full.reshape(-1)]))
        self.ptr = self.buf.ptr + 4 * shift

    def get(self):
        b, n, h, d = self.shape
        raw = self.buf.numpy()
        full = raw[self.shift:].reshape(b, n, self.ld)
        assert (raw[:self.shift] == 7.5).all() and (full[:, :, h * d:] == 7.5).all()  # nothing beside the tensor is written
        return full[:, :, :h * d].reshape(b, n, h, d)


class Case:
    def __init__(self, hip, batch, seq, heads, kv_heads, dim, window, sinks, lengths=None, pad=0, shift=0, acc=0, seed=0,
                 amp=(1, 1, 1, 1), spoil=None):
        r = rng(seed + 1000 * seq + dim)
        self.hip, self.dims = hip, (batch, seq, heads, kv_heads, dim)
        self.window, self.sinks, self.acc, self.scale = window, sinks, acc, ref.scale_of(dim)
        n = lambda h, a: (a * r.standard_normal((batch, seq, h, dim))).astype(np.float32)  # noqa: E731
        self.q, self.k, self.v, self.dout = n(heads, amp[0]), n(kv_heads, amp[1]), n(kv_heads, amp[2]), n(heads, amp[3])
        self.lengths = None if lengths is None else np.asarray(lengths, np.int32)
        if spoil:
            spoil(self)
        self.old = [n(heads, 1), n(kv_heads, 1), n(kv_heads, 1)]
        f = lambda a: Field(hip, a, pad, shift)  # noqa: E731
        self.gq, self.gk, self.gv, self.gdout = f(self.q), f(self.k), f(self.v), f(self.dout)
        self.out = f(np.full_like(self.q, np.nan))
        self.dq, self.dk, self.dv = (f(o) for o in self.old)
        self.lse = hip.Buffer.empty((batch, heads, seq))
        self.len = None if lengths is None else hip.Buffer.from_array(self.lengths)
        self.ws = hip.Buffer(hip.lib().mle_window_attention_ws_bytes(batch, seq, heads, kv_heads, dim, window, sinks))

    def forward(self, stream=None):
        b, n, h, kv, d = self.dims
        self.hip.call("mle_window_attention_fwd", stream, self.gq.ptr, self.gq.ld, self.gk.ptr, self.gk.ld, self.gv.ptr,
                      self.gv.ld, self.out.ptr, self.out.ld, self.lse.ptr, self.len.ptr if self.len else None, b, n, h, kv, d,
                      self.scale, self.window, self.sinks)

    def backward(self, stream=None):
        b, n, h, kv, d = self.dims
        a = self.acc
        self.hip.call("mle_window_attention_bwd", stream, self.gq.ptr, self.gq.ld, self.gk.ptr, self.gk.ld, self.gv.ptr,
                      self.gv.ld, self.out.ptr, self.out.ld, self.lse.ptr, self.gdout.ptr, self.gdout.ld, self.dq.ptr,
                      self.dq.ld, a & 1, self.dk.ptr, self.dk.ld, a & 2, self.dv.ptr, self.dv.ld, a & 4,
                      self.len.ptr if self.len else None, b, n, h, kv, d, self.scale, self.window, self.sinks, self.ws.ptr,
                      self.ws.nbytes)

    def results(self):
        return dict(out=self.out.get(), lse=self.lse.numpy(), dq=self.dq.get(), dk=self.dk.get(), dv=self.dv.get())

    def expected(self):
        b, n, h, kv, d = self.dims
        return ref.whole(self.q, self.k, self.v, self.lengths, h, kv, self.window, self.sinks, self.scale, self.dout)

    def check(self):
        got, r = self.results(), self.expected()
        for name in ("out", "lse"):
            ref.check(got[name], r, name)
        for i, name in enumerate(("dq", "dk", "dv")):
            ref.check(got[name], r, name, self.old[i] if self.acc >> i & 1 else None)
        return got


#        batch seq heads kv dim window sinks lengths pad shift acc
CASES = [
    (1, 1, 1, 1, 64, 1, 0, None, 0, 0, 0),
    (2, 2, 2, 1, 1, 2, 0, None, 0, 0, 7),
    (1, 17, 3, 3, 16, 5, 2, None, 0, 0, 0),
    (3, 33, 4, 2, 32, 33, 0, [33, 0, 1], 0, 0, 0),
    (2, 64, 4, 4, 64, 64, 0, None, 0, 0, 0),
    (2, 65, 2, 2, 64, 1, 1, None, 0, 0, 5),
    (1, 127, 6, 2, 128, 32, 4, None, 4, 0, 0),
    (2, 128, 2, 1, 64, 128, 0, [100, 128], 0, 0, 2),
    (2, 129, 4, 1, 40, 64, 64, [129, 7], 3, 1, 7),
    (1, 200, 2, 2, 31, 63, 70, None, 1, 1, 0),
    (2, 257, 8, 2, 64, 100, 4, [257, 130], 0, 0, 0),
    (1, 300, 2, 2, 80, 1000, 3, None, 0, 0, 0),
    (3, 333, 6, 2, 96, 50, 0, [333, 0, 64], 0, 0, 0),
    (1, 640, 4, 4, 64, 129, 33, None, 0, 0, 4),
    (2, 1100, 4, 2, 64, 96, 5, [1100, 1001], 0, 0, 0),
    (1, 1500, 2, 1, 128, 300, 130, None, 0, 0, 0),
    (1, 2500, 1, 1, 64, 2500, 0, None, 0, 0, 0),
    (70, 40, 2, 1, 24, 9, 2, None, 0, 0, 0),
    (1, 600, 12, 3, 127, 200, 1, None, 2, 3, 3),
]


# many heads: every number of waves and of key blocks that the launches choose from, at each width
CASES += [
    (40, 140, 8, 4, 64, 60, 2, None, 0, 0, 0),
    (24, 150, 6, 6, 90, 70, 3, [150, 0, 1, 149, 128, 33] * 4, 0, 0, 0),
    (20, 131, 8, 2, 128, 40, 0, None, 0, 0, 7),
    (32, 40, 8, 8, 64, 600, 1, [40, 3] * 16, 0, 0, 2),
    (16, 300, 8, 4, 128, 512, 0, None, 0, 0, 0),
    (32, 33, 8, 1, 72, 512, 2, None, 1, 2, 0),
    (16, 200, 5, 5, 64, 50, 1, None, 0, 0, 0),
    (16, 129, 6, 3, 96, 300, 0, [129, 128, 65, 64] * 4, 0, 0, 0),
    (12, 256, 8, 8, 128, 90, 2, None, 0, 0, 0),
    (1, 3, 300, 100, 5, 2, 1, None, 0, 0, 0),
    (1, 1500, 2, 2, 32, 3, 1400, [1499], 0, 0, 2),
    (2, 900, 4, 2, 100, 1, 900, [900, 40], 0, 0, 0),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace(" ", "") for x in c))
def test_forward_and_backward(hip, case):
    b, n, h, kv, d, w, s, lengths, pad, shift, acc = case
    c = Case(hip, b, n, h, kv, d, w, s, lengths, pad, shift, acc)
    c.forward()
    c.backward()
    c.check()


@pytest.mark.parametrize("amp", [(1e-20, 1e20, 1, 1), (3, 3, 1e15, 1e-25), (1, 1, 1e-30, 1e10), (6, 6, 1, 1e-8), (1e-3, 1e-3, 1, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_sizes_of_values(hip, amp, dim):
    """Tensors of any size of values, and scores from even to one-sided."""
    c = Case(hip, 1, 300, 2, 1, dim, 120, 3, amp=amp)
    c.forward()
    c.backward()
    c.check()


def test_rows_of_unlike_size(hip):
    """A token's rows may be far larger than its neighbours': each key's and each query's gradient keeps its bits."""
    def spoil(c):
        r = rng(9)
        for a in (c.v, c.dout):
            a *= (10.0 ** r.uniform(-4, 0, a.shape[:2] + (1, 1))).astype(np.float32)
    c = Case(hip, 2, 400, 4, 2, 64, 150, 4, spoil=spoil)
    c.forward()
    c.backward()
    c.check()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_what_the_window_has_left_may_be_large(hip, which, dim):
    """Entries 2^30 times the others' that a row no longer sees cost it no bits."""
    small, large = Case(hip, 1, 400, 4, 2, dim, 40, 0), Case(
        hip, 1, 400, 4, 2, dim, 40, 0, spoil=lambda c: getattr(c, which).__setitem__((0, slice(0, 60)), getattr(c, which)[0, :60] * np.float32(2 ** 30)))
    for c in (small, large):
        c.forward()
        c.backward()
    r, got = small.expected(), large.results()
    at = slice(192, None)  # tiles after the large ones' and the window's
    for name in ("out", "dq", "dk", "dv"):
        ref.check(got[name][:, at], {name: r[name][:, at], "e_" + name: r["e_" + name][:, at]}, name)
    ref.check(got["lse"][:, :, at], {"lse": r["lse"][:, :, at], "e_lse": r["e_lse"][:, :, at]}, "lse")


@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-6])
@pytest.mark.parametrize("dim", [48, 120])
def test_scales(hip, scale, dim):
    c = Case(hip, 2, 150, 4, 2, dim, 60, 2, lengths=[150, 90])
    c.scale = float(np.float32(scale))
    c.forward()
    c.backward()
    c.check()


def test_what_is_hidden_may_hold_anything(hip):
    """Rows past a length (NaN, infinities, the largest numbers) reach nothing, and their gradients are 0."""
    def spoil(c):
        for b, n in enumerate(c.lengths):
            for i, a in enumerate((c.q, c.k, c.v, c.dout)):
                a[b, n:] = (np.nan, np.inf, -np.inf, 3e38)[i]
                a[b, n:, :, ::2] = np.nan
    c = Case(hip, 3, 290, 4, 2, 64, 70, 4, [290, 131, 0], spoil=spoil)
    c.forward()
    c.backward()
    got = c.check()
    for b, n in enumerate(c.lengths):
        for name in ("out", "dq", "dk", "dv"):
            assert (got[name][b, n:] == 0).all(), name


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("which", ["q", "k", "v", "dout"])
def test_one_entry_that_is_not_finite(hip, which, value):
    """An entry that is not finite reaches the rows and keys that see it, and no others."""
    n, w, s, at = 260, 40, 2, 100
    def spoil(c):
        getattr(c, which)[0, at, 0, 5] = value
    c = Case(hip, 1, n, 2, 1, 64, w, s, spoil=spoil)
    c.forward()
    c.backward()
    got = c.results()
    clean = Case(hip, 1, n, 2, 1, 64, w, s)
    r = clean.expected()
    i = np.arange(n)
    rows = {"q": i == at, "dout": i == at, "k": (i >= at) & (i < at + w), "v": (i >= at) & (i < at + w)}[which]
    heads = [0] if which in ("q", "dout") else [0, 1]
    hit = np.zeros((n, 2), bool)
    hit[np.ix_(np.nonzero(rows)[0], heads)] = True
    if which != "dout":
        assert np.isfinite(got["out"][0][~hit]).all()
        err = np.abs(got["out"] - r["out"])[0][~hit]
        assert (err <= r["e_out"][0][~hit]).all()
        if which in ("q", "k") and np.isnan(value):
            assert np.isnan(got["out"][0][hit]).all()
        if which == "v":
            assert not np.isfinite(got["out"][0][hit][:, 5]).any() and np.isfinite(np.delete(got["out"][0][hit], 5, 1)).all()
    err = np.abs(got["dq"] - r["dq"])[0][~hit]
    assert (err <= r["e_dq"][0][~hit]).all()
    # keys that no query seeing the entry sees
    see = ref.visible(i, n, w, s)
    free = ~see[hit.any(1)].any(0)
    for name in ("dk", "dv"):
        assert (np.abs(got[name] - r[name])[0][free] <= r["e_" + name][0][free]).all(), name
    if which in ("k", "v"):
        assert not np.isfinite(got["dq"][0][hit]).all()


def test_gradient_against_differences(hip):
    """dq, dk and dv against central differences of <out, dout> of the 64-bit formula."""
    c = Case(hip, 1, 70, 2, 1, 24, 20, 3)
    c.forward()
    c.backward()
    got = c.results()

    def f(q, k, v):
        total = 0.0
        for h in range(2):
            see = ref.visible(np.arange(70), 70, 20, 3)
            x = np.where(see, c.scale * (q[0, :, h] @ k[0, :, 0].T), -np.inf)
            p = np.exp(x - x.max(1, keepdims=True))
            total += float((p / p.sum(1, keepdims=True) @ v[0, :, 0] * c.dout[0, :, h]).sum())
        return total

    x = [a.astype(np.float64) for a in (c.q, c.k, c.v)]
    step = 1e-5
    for t, name in enumerate(("dq", "dk", "dv")):
        for i, d in ((0, 0), (1, 7), (40, 23), (69, 11)):
            at = (0, i, x[t].shape[2] - 1, d)
            y = [a.copy() for a in x]
            y[t][at] += step
            up = f(*y)
            y[t][at] -= 2 * step
            assert abs((up - f(*y)) / (2 * step) - got[name][at]) <= 1e-4, (name, at)


def test_same_bits_twice_and_without_lse(hip):
    c = Case(hip, 2, 500, 4, 2, 64, 130, 4, [500, 301])
    c.forward()
    c.backward()
    one = c.results()
    c.forward()
    c.backward()
    two = c.results()
    for name in one:
        assert np.array_equal(one[name], two[name]), name
    b, n, h, kv, d = c.dims
    hip.call("mle_window_attention_fwd", None, c.gq.ptr, c.gq.ld, c.gk.ptr, c.gk.ld, c.gv.ptr, c.gv.ld, c.out.ptr, c.out.ld,
             None, c.len.ptr, b, n, h, kv, d, c.scale, c.window, c.sinks)
    assert np.array_equal(c.out.get(), one["out"])


def test_offsets_past_32_bits(hip):
    """Rows a gigabyte apart."""
    n, d, ld = 9, 64, 1 << 28
    r = rng(3)
    x = r.standard_normal((8, n, d)).astype(np.float32)  # q k v out dout dq dk dv side by side
    big = hip.Buffer(4 * ((n - 1) * ld + 8 * d))
    for t in range(8):
        for i in range(n):
            hip.call("mle_memcpy_h2d", big.ptr + 4 * (i * ld + t * d), x[t, i].ctypes.data, 4 * d, None)
    p = [big.ptr + 4 * t * d for t in range(8)]
    lse, ws = hip.Buffer.empty((1, 1, n)), hip.Buffer(hip.lib().mle_window_attention_ws_bytes(1, n, 1, 1, d, 4, 1))
    sc = ref.scale_of(d)
    hip.call("mle_window_attention_fwd", None, p[0], ld, p[1], ld, p[2], ld, p[3], ld, lse.ptr, None, 1, n, 1, 1, d, sc, 4, 1)
    hip.call("mle_window_attention_bwd", None, p[0], ld, p[1], ld, p[2], ld, p[3], ld, lse.ptr, p[4], ld, p[5], ld, 0, p[6], ld,
             0, p[7], ld, 0, None, 1, n, 1, 1, d, sc, 4, 1, ws.ptr, ws.nbytes)
    hip.sync()
    got = np.empty((8, n, d), np.float32)
    for t in range(8):
        for i in range(n):
            hip.call("mle_memcpy_d2h", got[t, i].ctypes.data, big.ptr + 4 * (i * ld + t * d), 4 * d, None)
    f = lambda a: a.reshape(1, n, 1, d)  # noqa: E731
    w = ref.whole(f(x[0]), f(x[1]), f(x[2]), None, 1, 1, 4, 1, sc, f(x[4]))
    for t, name in ((3, "out"), (5, "dq"), (6, "dk"), (7, "dv")):
        ref.check(f(got[t]), w, name)
    length = hip.Buffer.from_array(np.array([n], np.int32))
    ws = hip.Buffer(max(16, hip.lib().mle_window_attention_step_ws_bytes(1, 1, n, 1, 1, d, 4, 1)))
    out = hip.Buffer.empty((1, 1, 1, d))
    hip.call("mle_window_attention_step", None, p[0] + 4 * (n - 1) * ld, ld, p[1], ld, p[2], ld, out.ptr, d, length.ptr, 1, 1,
             n, 1, 1, d, sc, 4, 1, ws.ptr, ws.nbytes)
    w = ref.whole(f(x[0])[:, n - 1:], f(x[1]), f(x[2]), [n], 1, 1, 4, 1, sc, at_end=True)
    ref.check(out.numpy(), w, "out")


# ------------------------------------------------------------- newest tokens


class Step:
    def __init__(self, hip, batch, tokens, cap, heads, kv_heads, dim, window, sinks, lengths, pad=0, shift=0, spoil=None,
                 amp=1.0):
        r = rng(cap + 7 * dim + tokens)
        self.hip, self.dims, self.window, self.sinks, self.scale = hip, (batch, tokens, cap, heads, kv_heads, dim), window, sinks, ref.scale_of(dim)
        self.q = (amp * r.standard_normal((batch, tokens, heads, dim))).astype(np.float32)
        self.k, self.v = (r.standard_normal((batch, cap, kv_heads, dim)).astype(np.float32) for _ in range(2))
        self.lengths = np.asarray(lengths, np.int32)
        if spoil:
            spoil(self)
        f = lambda a: Field(hip, a, pad, shift)  # noqa: E731
        self.gq, self.gk, self.gv, self.out = f(self.q), f(self.k), f(self.v), f(np.full_like(self.q, np.nan))
        self.len = hip.Buffer.from_array(self.lengths)
        self.ws = hip.Buffer(max(16, hip.lib().mle_window_attention_step_ws_bytes(batch, tokens, cap, heads, kv_heads, dim, window, sinks)))

    def run(self, stream=None):
        b, t, cap, h, kv, d = self.dims
        self.hip.call("mle_window_attention_step", stream, self.gq.ptr, self.gq.ld, self.gk.ptr, self.gk.ld, self.gv.ptr,
                      self.gv.ld, self.out.ptr, self.out.ld, self.len.ptr, b, t, cap, h, kv, d, self.scale, self.window,
                      self.sinks, self.ws.ptr, self.ws.nbytes)

    def expected(self):
        b, t, cap, h, kv, d = self.dims
        return ref.whole(self.q, self.k, self.v, self.lengths, h, kv, self.window, self.sinks, self.scale, at_end=True)

    def check(self):
        got = self.out.get()
        ref.check(got, self.expected(), "out")
        return got


#        batch tokens cap heads kv dim window sinks lengths pad shift
STEPS = [
    (1, 1, 1, 1, 1, 64, 1, 0, [1], 0, 0),
    (3, 1, 40, 4, 2, 16, 7, 2, [40, 1, 0], 0, 0),
    (2, 1, 64, 8, 8, 64, 128, 4, [64, 33], 0, 0),
    (4, 1, 500, 8, 2, 128, 200, 4, [500, 499, 204, 3], 0, 0),
    (2, 1, 3000, 4, 1, 128, 2000, 5, [3000, 2222], 0, 0),
    (2, 1, 3000, 6, 2, 80, 5000, 0, [2999, 17], 0, 0),
    (1, 1, 5000, 32, 1, 64, 300, 40, [4999], 0, 0),
    (2, 3, 700, 12, 3, 40, 100, 70, [700, 2], 3, 1),
    (3, 5, 300, 8, 4, 33, 16, 1, [300, 5, 4], 1, 3),
    (1, 40, 600, 8, 2, 64, 128, 4, [555], 0, 0),
    (2, 16, 16, 2, 1, 127, 16, 0, [16, 9], 0, 0),
    (1, 300, 1000, 4, 2, 128, 200, 3, [900], 0, 0),
    (2, 1, 20, 3, 3, 1, 5, 1, [25, -3], 0, 0),   # lengths past the capacity and below 0
    (70, 2, 90, 2, 2, 32, 30, 2, list(range(1, 71)), 0, 0),
]


@pytest.mark.parametrize("case", STEPS, ids=lambda c: "-".join(str(x) for x in c[:8]))
def test_newest_tokens(hip, case):
    s = Step(hip, *case)
    s.run()
    s.check()


def test_newest_tokens_and_what_is_hidden(hip):
    """The cache past a length and between the sinks and the window may hold anything."""
    def spoil(s):
        s.k[0, 900:] = np.nan
        s.v[0, 900:] = np.inf
        s.k[0, 5:600] = -np.inf
        s.v[0, 5:600] = np.nan
        s.k[1, 77:] = s.v[1, 77:] = np.nan
    s = Step(hip, 2, 1, 1000, 8, 2, 64, 300, 5, [900, 77], spoil=spoil)
    s.run()
    assert np.isfinite(s.check()).all()


def test_newest_tokens_seeing_nan_and_large_scores(hip):
    s = Step(hip, 2, 1, 800, 4, 2, 64, 500, 2, [800, 600], amp=30.0)
    s.run()
    s.check()
    def spoil(s):
        s.v[0, 700, 1, 3] = np.nan
        s.k[1, 500, 0, 0] = np.nan
    s = Step(hip, 2, 1, 800, 4, 2, 64, 500, 2, [800, 600], spoil=spoil)
    s.run()
    got = s.out.get()
    assert np.isnan(got[0, 0, 2:, 3]).all() and np.isfinite(np.delete(got[0, 0], 3, 1)).all() and np.isfinite(got[0, 0, :2]).all()
    assert np.isnan(got[1, 0, :2]).all() and np.isfinite(got[1, 0, 2:]).all()


def test_step_agrees_with_the_whole_pass(hip):
    """Token by token over a cache gives what the pass over the sequence gives, to their bounds."""
    c = Case(hip, 1, 150, 4, 2, 64, 40, 3)
    c.forward()
    r = c.expected()
    for p in (0, 1, 39, 40, 44, 100, 149):
        s = Step(hip, 1, 1, 150, 4, 2, 64, 40, 3, [p + 1])
        s.k, s.v, s.q = c.k, c.v, c.q[:, p:p + 1]
        s.gk, s.gv, s.gq = (Field(hip, a) for a in (s.k, s.v, np.ascontiguousarray(s.q)))
        s.run()
        got = s.check()
        assert (np.abs(got - c.out.get()[:, p:p + 1]) <= 2 * r["e_out"][:, p:p + 1]).all()


# ---------------------------------------------------------- streams and graphs


def test_captured_and_replayed(hip):
    """The recorded calls, replayed between eager work on other data, give the eager calls' bits."""
    st, graph = C.c_void_p(), C.c_void_p()
    hip.call("mle_stream_create", C.byref(st))
    c, s = Case(hip, 2, 300, 4, 2, 64, 100, 4, [300, 177]), Step(hip, 2, 1, 900, 4, 2, 64, 500, 3, [900, 600])
    hip.call("mle_graph_capture_begin", st)
    c.forward(st)
    c.backward(st)
    s.run(st)
    hip.call("mle_graph_capture_end", st, C.byref(graph))
    other = Case(hip, 1, 200, 2, 2, 128, 50, 2)
    for turn in range(3):
        q = rng(50 + turn).standard_normal(c.q.shape).astype(np.float32)
        c.q[:] = q
        c.gq.buf.upload(q.reshape(-1))
        hip.call("mle_graph_launch", graph, st)
        hip.sync(st)
        replayed, token = c.results(), s.out.get()
        other.forward()
        other.backward()
        other.check()
        c.forward()
        c.backward()
        s.run()
        hip.sync()
        for name, a in c.results().items():
            assert np.array_equal(a, replayed[name]), (turn, name)
        assert np.array_equal(token, s.out.get())
        c.check()
    hip.call("mle_graph_destroy", graph)
    hip.call("mle_stream_destroy", st)


def test_two_streams(hip):
    """Calls at once on two streams, each with its own workspace."""
    st = [C.c_void_p() for _ in range(2)]
    for x in st:
        hip.call("mle_stream_create", C.byref(x))
    cases = [Case(hip, 1, 700, 4, 2, 64, 200, 4), Case(hip, 2, 400, 4, 4, 128, 100, 40)]
    steps = [Step(hip, 3, 1, 2000, 8, 2, 64, 1500, 3, [2000, 1700, 5]), Step(hip, 1, 1, 4000, 8, 1, 128, 4000, 0, [4000])]
    for _ in range(3):
        for x, c, s in zip(st, cases, steps):
            c.forward(x)
            c.backward(x)
            s.run(x)
    for x in st:
        hip.sync(x)
    for c, s in zip(cases, steps):
        c.check()
        s.check()
    for x in st:
        hip.call("mle_stream_destroy", x)


def test_nothing_to_do(hip):
    hip.call("mle_window_attention_fwd", None, None, 64, None, 64, None, 64, None, 64, None, None, 0, 8, 1, 1, 64, 1.0, 4, 0)
    hip.call("mle_window_attention_bwd", None, None, 64, None, 64, None, 64, None, 64, None, None, 64, None, 64, 0, None, 64, 0,
             None, 64, 0, None, 2, 0, 1, 1, 64, 1.0, 4, 0, None, 0)
    hip.call("mle_window_attention_step", None, None, 64, None, 64, None, 64, None, 64, None, 2, 0, 8, 1, 1, 64, 1.0, 4, 0, None, 0)
    out = hip.Buffer.from_array(np.full((2, 3, 64), 5, np.float32))  # an empty cache: rows without a key
    q, n = hip.Buffer.zeros((2, 3, 64)), hip.Buffer.zeros(2, np.int32)
    hip.call("mle_window_attention_step", None, q.ptr, 64, None, 64, None, 64, out.ptr, 64, n.ptr, 2, 3, 0, 1, 1, 64, 1.0, 4, 0,
             None, 0)
    assert (out.numpy() == 0).all()
