"""The vocabulary cross entropy, the 8-bit checkpoints, the norm with 8-bit output
and the scaled embedding run together, as one training pass of a small language
model through the C entry points: against 64 bits, on another stream, two passes on
two streams at once, and replayed from a recorded graph."""
import math

import numpy as np
import pytest

import q8_ref
from conftest import rng

pytestmark = pytest.mark.gpu
EPS = 1e-5


class Pass:
    """h0 = s E[ids]; y = norm(h0), kept in 8 bits; u = y W1 + b1, kept in 8 bits;
    a = gelu(u); r = a W2; z = norm(h0 + r), and the vocabulary's cross entropy of z.  The
    backward reads y and u from their 8 bits."""

    def __init__(self, hip, B, S, D, F, V, seed=0):
        r = rng(seed)
        self.hip, self.dims = hip, (B, S, D, F, V)
        T = B * S
        u = lambda *s, b: r.uniform(-b, b, s).astype(np.float32)  # noqa: E731
        self.p = dict(E=u(V, D, b=0.2), n1=1 + u(D, b=0.2), W1=u(D, F, b=math.sqrt(3 / D)), b1=u(F, b=0.1),
                      W2=u(F, D, b=math.sqrt(3 / F)), n2=1 + u(D, b=0.2), W=u(D, V, b=math.sqrt(3 / D)), b=u(V, b=0.1))
        self.ids, self.tgt = (r.integers(0, V, (B, S)).astype(np.int32) for _ in range(2))
        self.ids[0, S - 5:] = -1
        self.tgt[0, S - 6:] = -1
        self.count = int((self.tgt >= 0).sum())
        Bf, L = hip.Buffer, hip.lib()
        self.d = {k: Bf.from_array(v) for k, v in self.p.items()}
        self.g = {k: Bf.empty(v.shape) for k, v in self.p.items()}
        self.dids, self.dtgt = Bf.from_array(self.ids), Bf.from_array(self.tgt)
        f = lambda *s: Bf.empty(s)  # noqa: E731
        self.h0, self.y, self.u, self.a, self.r, self.h1, self.z = f(T, D), f(T, D), f(T, F), f(T, F), f(T, D), f(T, D), f(T, D)
        self.s1, self.s2, self.lse, self.loss = f(T), f(T), f(T), f(1)
        self.dz, self.dh1, self.da, self.du, self.dy, self.dh0 = f(T, D), f(T, D), f(T, F), f(T, F), f(T, D), f(T, D)
        self.gd, self.gf = -(-D // 32), -(-F // 32)
        self.qy, self.ey = Bf.empty((T, D), np.int8), Bf.empty((T, self.gd), np.uint8)
        self.qu, self.eu = Bf.empty((T, F), np.int8), Bf.empty((T, self.gf), np.uint8)
        self.ix = Bf(L.mle_embed_sorted_index_bytes(B, S, V))
        need = max(L.mle_vocab_xent_ws_bytes(T, D, V), L.mle_q8_linear_wgrad_ws_bytes(T, D, F), L.mle_add_rmsnorm_ws_bytes(T, D),
                   L.mle_embed_sorted_grad_ws_bytes(B, S, D), L.mle_linear_bwd_ws_bytes(T, F, D, 1), L.mle_gemm_ws_bytes(T, F, D, 1),
                   L.mle_gemm_ws_bytes(T, D, F, 1))
        self.ws = Bf(need)

    def run(self, s=None):
        """One pass: one workspace serves every call, in the stream's order."""
        B, S, D, F, V = self.dims
        T, call, d, g, ws = B * S, self.hip.call, self.d, self.g, (self.ws.ptr, self.ws.nbytes)
        gelu, scale = self.hip.ACT["gelu"], math.sqrt(D)
        call("mle_embed_scaled_fwd", s, self.h0.ptr, d["E"].ptr, self.dids.ptr, B, S, S, D, V, scale, self.ix.ptr, self.ix.nbytes)
        call("mle_add_rmsnorm_q8_fwd", s, T, D, self.h0.ptr, None, d["n1"].ptr, EPS, None, self.y.ptr, self.s1.ptr, self.qy.ptr,
             D, self.ey.ptr, self.gd)
        call("mle_gemm_ex", s, 0, 0, T, F, D, 1.0, self.y.ptr, D, 0, d["W1"].ptr, F, 0, 0.0, self.u.ptr, F, 0, 1, None,
             d["b1"].ptr, *ws)
        call("mle_q8_act_fwd", s, gelu, T, F, self.u.ptr, F, self.a.ptr, F, self.qu.ptr, F, self.eu.ptr, self.gf)
        call("mle_gemm_ex", s, 0, 0, T, D, F, 1.0, self.a.ptr, F, 0, d["W2"].ptr, D, 0, 0.0, self.r.ptr, D, 0, 1, None, None, *ws)
        call("mle_add_rmsnorm_q8_fwd", s, T, D, self.h0.ptr, self.r.ptr, d["n2"].ptr, EPS, self.h1.ptr, self.z.ptr, self.s2.ptr,
             None, 0, None, 0)
        loss = (T, D, V, self.z.ptr, D, d["W"].ptr, V, d["b"].ptr, self.dtgt.ptr, S, S)
        call("mle_vocab_xent_fwd", s, *loss, 1.0 / self.count, self.lse.ptr, None, self.loss.ptr, *ws)

        call("mle_vocab_xent_bwd", s, *loss, self.lse.ptr, None, 1.0 / self.count, self.dz.ptr, D, 0, g["W"].ptr, V, g["b"].ptr,
             0, *ws)
        call("mle_add_rmsnorm_bwd", s, T, D, self.h1.ptr, d["n2"].ptr, self.s2.ptr, self.dz.ptr, None, self.dh1.ptr, 0,
             g["n2"].ptr, 0, *ws)
        call("mle_linear_bwd_ex", s, T, F, D, 1, self.a.ptr, self.dh1.ptr, 0, d["W2"].ptr, 0, self.da.ptr, 0, g["W2"].ptr, None,
             0, 0, *ws)
        call("mle_q8_act_bwd", s, gelu, T, F, self.qu.ptr, F, self.eu.ptr, self.gf, self.da.ptr, F, self.du.ptr, F, 0)
        call("mle_q8_linear_wgrad", s, T, D, F, self.qy.ptr, D, self.ey.ptr, self.gd, self.du.ptr, F, g["W1"].ptr, F,
             g["b1"].ptr, 0, *ws)
        call("mle_gemm_ex", s, 0, 1, T, D, F, 1.0, self.du.ptr, F, 0, d["W1"].ptr, F, 0, 0.0, self.dy.ptr, D, 0, 1, None, None, *ws)
        call("mle_add_rmsnorm_bwd", s, T, D, self.h0.ptr, d["n1"].ptr, self.s1.ptr, self.dy.ptr, self.dh1.ptr, self.dh0.ptr, 0,
             g["n1"].ptr, 0, *ws)
        call("mle_embed_sorted_grad", s, g["E"].ptr, self.dh0.ptr, self.ix.ptr, self.ix.nbytes, B, S, D, V, scale, 0, *ws)

    def results(self):
        return dict(loss=self.loss.numpy(), **{k: v.numpy() for k, v in self.g.items()})

    def exact(self):
        """In 64 bits, from the kept 8 bits of the device's own y and u."""
        B, S, D, F, V = self.dims
        p = {k: v.astype(np.float64) for k, v in self.p.items()}
        k, t = self.ids.reshape(-1), self.tgt.reshape(-1)
        ok, tk, scale = k >= 0, t >= 0, float(np.float32(math.sqrt(D)))
        h0 = np.where(ok[:, None], p["E"][np.maximum(k, 0)], 0) * scale
        norm = lambda h: 1 / np.sqrt((h * h).mean(1, keepdims=True) + EPS)  # noqa: E731
        s1 = norm(h0)
        y = h0 * s1 * p["n1"]
        u = y @ p["W1"] + p["b1"]
        c = math.sqrt(2 / math.pi)
        a = 0.5 * u * (1 + np.tanh(c * (u + 0.044715 * u ** 3)))
        h1 = h0 + a @ p["W2"]
        s2 = norm(h1)
        z = h1 * s2 * p["n2"]
        l = z @ p["W"] + p["b"]
        l -= l.max(1, keepdims=True)
        pr = np.exp(l)
        pr /= pr.sum(1, keepdims=True)
        at, tt = np.arange(B * S), np.where(tk, t, 0)
        loss = -(np.log(pr[at, tt]) * tk).sum() / self.count
        pr[at, tt] -= 1
        pr *= tk[:, None] / self.count
        dz = pr @ p["W"].T

        def back(h, s, w, dout):
            v, gr = h * s, dout * w
            return s * (gr - v * (gr * v).mean(1, keepdims=True)), (dout * v).sum(0)

        dh1, dn2 = back(h1, s2, p["n2"], dz)
        ku = q8_ref.kept(self.u.numpy()).astype(np.float64)
        th = np.tanh(c * (ku + 0.044715 * ku ** 3))
        du = (dh1 @ p["W2"].T) * (0.5 * (1 + th) + 0.5 * ku * (1 - th ** 2) * c * (1 + 0.134145 * ku ** 2))
        ky = q8_ref.kept(self.y.numpy()).astype(np.float64)
        dh0, dn1 = back(h0, s1, p["n1"], du @ p["W1"].T)
        dh0 += dh1
        dE = np.zeros_like(p["E"])
        np.add.at(dE, k[ok], dh0[ok] * scale)
        return dict(loss=np.array([loss]), E=dE, n1=dn1, W1=ky.T @ du, b1=du.sum(0), W2=a.T @ dh1, n2=dn2, W=z.T @ pr, b=pr.sum(0))


SHAPES = [(2, 30, 48, 72, 211), (3, 150, 64, 130, 1003), (1, 400, 96, 64, 20000)]


@pytest.mark.parametrize("shape", SHAPES)
def test_pass(hip, shape):
    m = Pass(hip, *shape)
    m.run()
    got, want = m.results(), m.exact()
    for k, w in want.items():
        # chains of fp32 sums: some 1e-6 of a tensor's largest value
        assert np.abs(got[k] - w).max() <= 1e-5 * np.abs(w).max(), k
    m.run()
    for k, w in m.results().items():
        assert np.array_equal(w, got[k]), k


def test_two_streams(hip):
    """Two passes at once, each on a stream and workspace of its own, give what they give alone."""
    passes = [Pass(hip, *SHAPES[1], seed=s) for s in (1, 2)]
    alone = []
    for m in passes:
        m.run()
        alone.append(m.results())
    streams = []
    for _ in passes:
        s = hip.P()
        hip.call("mle_stream_create", hip.C.byref(s))
        streams.append(s.value)
    for m in passes:
        for b in m.g.values():
            b.upload(np.full(b.shape, np.nan, np.float32))
    hip.sync()
    for _ in range(3):
        for m, s in zip(passes, streams):
            m.run(s)
    for s in streams:
        hip.sync(s)
    for m, want in zip(passes, alone):
        for k, v in m.results().items():
            assert np.array_equal(v, want[k]), k
    for s in streams:
        hip.call("mle_stream_destroy", s)


@pytest.mark.parametrize("shape", SHAPES[:2])
def test_replayed(hip, shape):
    """A recorded pass replayed with other parameters and ids, between eager passes."""
    m, other = Pass(hip, *shape), Pass(hip, *shape, seed=7)
    m.run()
    first = m.results()
    s, g = hip.P(), hip.P()
    hip.call("mle_stream_create", hip.C.byref(s))
    hip.call("mle_graph_capture_begin", s.value)
    m.run(s.value)
    hip.call("mle_graph_capture_end", s.value, hip.C.byref(g))
    other.run()
    want = other.results()
    assert m.count == other.count  # (the scale is recorded)
    for turn in range(4):
        src, ref = ((m.p, m.ids, m.tgt), first) if turn % 2 == 0 else ((other.p, other.ids, other.tgt), want)
        for k, v in src[0].items():
            m.d[k].upload(v)
        m.dids.upload(src[1])
        m.dtgt.upload(src[2])
        hip.sync()
        hip.call("mle_graph_launch", g.value, s.value)
        hip.sync(s.value)
        for k, v in m.results().items():
            assert np.array_equal(v, ref[k]), (turn, k)
        other.run()
        hip.sync()
        assert np.array_equal(other.loss.numpy(), want["loss"])
    hip.call("mle_graph_destroy", g.value)
    hip.call("mle_stream_destroy", s.value)
