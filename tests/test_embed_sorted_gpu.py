"""Scaled embedding lookup (equal bit for bit) and the table's gradient by
sorted tokens (against 64 bits)."""
import numpy as np
import pytest

from conftest import rng

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -24  # half a step of fp32


def forward(hip, keys, table, clen, scale, shift=0, stream=None):
    batch, max_clen = keys.shape
    vocab, dim = table.shape
    gk = hip.Buffer.from_array(np.concatenate([np.zeros(shift, np.int32), keys.reshape(-1)]))
    gt = hip.Buffer.from_array(np.concatenate([np.zeros(shift, np.float32), table.reshape(-1)]))
    go = hip.Buffer.from_array(np.full(batch * clen * dim + 8, 5.0, np.float32))
    ix = hip.Buffer(hip.lib().mle_embed_sorted_index_bytes(batch, clen, vocab))
    hip.call("mle_embed_scaled_fwd", stream, go.ptr, gt.ptr + 4 * shift, gk.ptr + 4 * shift, batch, clen, max_clen, dim, vocab, scale,
             ix.ptr, ix.nbytes)
    out = go.numpy()
    assert (out[batch * clen * dim:] == 5.0).all()
    return out[: batch * clen * dim].reshape(batch, clen, dim), ix


def gradient(hip, ix, dy, vocab, scale, acc, old, shift=0, stream=None):
    batch, clen, dim = dy.shape
    gd = hip.Buffer.from_array(np.concatenate([np.zeros(shift, np.float32), dy.reshape(-1)]))
    gt = hip.Buffer.from_array(np.concatenate([old.reshape(-1), np.full(8, 5.0, np.float32)]))
    ws = hip.Buffer(hip.lib().mle_embed_sorted_grad_ws_bytes(batch, clen, dim))
    hip.call("mle_embed_sorted_grad", stream, gt.ptr, gd.ptr + 4 * shift, ix.ptr, ix.nbytes, batch, clen, dim, vocab, scale,
             acc, ws.ptr, ws.nbytes)
    t = gt.numpy()
    assert (t[vocab * dim:] == 5.0).all()
    return t[: vocab * dim].reshape(vocab, dim)


def ids(r, kind, batch, clen, max_clen, vocab):
    n = batch * max_clen
    if kind == "uniform":
        k = r.integers(0, vocab, n)
    elif kind == "frequent":
        k = np.minimum(np.exp(r.random(n) * np.log(vocab + 1.0)).astype(np.int64) - 1, vocab - 1)
    elif kind == "one":
        k = np.full(n, vocab // 2)
    else:  # "outside": negative, past the vocabulary, INT_MIN among ordinary ones
        k = r.choice(np.array([-1, -2 ** 31, vocab, 2 ** 31 - 1, 0, vocab - 1]), n)
    k = k.astype(np.int32).reshape(batch, max_clen)
    k[:, clen:] = vocab - 1  # never read
    return k


CASES = [("uniform", 1, 1, 1, 1, 1), ("uniform", 1, 1, 3, 50, 7), ("uniform", 2, 17, 20, 50, 33), ("frequent", 4, 100, 100, 1000, 48),
         ("one", 3, 40, 41, 9, 64), ("one", 1, 17, 17, 5, 260), ("one", 2, 5000, 5000, 40000, 16), ("outside", 5, 30, 30, 20, 32),
         ("frequent", 8, 256, 256, 8000, 512), ("frequent", 3, 3000, 3001, 33000, 100), ("uniform", 4, 4500, 4500, 300, 20),
         ("frequent", 2, 500, 512, 128000, 200), ("uniform", 1, 300, 300, 600000, 4), ("uniform", 1, 16, 16, 1, 2052),
         ("one", 1, 16, 16, 3, 12), ("frequent", 1, 9000, 9000, 17, 1030),
         # rows whose last four columns reach into the group before
         ("frequent", 5, 200, 200, 40, 5), ("frequent", 5, 200, 203, 300, 6), ("one", 2, 300, 300, 7, 7),
         ("frequent", 4, 300, 301, 90, 1031), ("uniform", 2, 40, 40, 30, 3),
         # several index workgroups to a range of rows
         ("frequent", 9, 4000, 4001, 300, 8), ("frequent", 4, 10000, 10000, 40000, 8), ("uniform", 2, 10001, 10001, 500, 520)]


@pytest.mark.parametrize("kind,batch,clen,max_clen,vocab,dim", CASES)
@pytest.mark.parametrize("acc,shift", [(0, 0), (1, 1)])
def test_lookup_and_gradient(hip, kind, batch, clen, max_clen, vocab, dim, acc, shift):
    r = rng(vocab + dim)
    keys, scale = ids(r, kind, batch, clen, max_clen, vocab), np.float32(np.sqrt(dim))
    table = r.standard_normal((vocab, dim)).astype(np.float32)
    dy = r.standard_normal((batch, clen, dim)).astype(np.float32)
    old = r.standard_normal((vocab, dim)).astype(np.float32)
    out, ix = forward(hip, keys, table, clen, scale, shift)
    k = keys[:, :clen].reshape(-1)
    ok = (k >= 0) & (k < vocab)
    ref = np.zeros((batch * clen, dim), np.float32)
    ref[ok] = table[k[ok]] * scale
    assert np.array_equal(out.reshape(-1, dim), ref)
    # the index: every token once, by id and then by place
    ints = ix.numpy(dtype=np.int32)
    n = int(ok.sum())
    assert ints[0] == n
    info = ints[64: 64 + 2 * vocab].reshape(vocab, 2)
    order = np.argsort(k[ok], kind="stable")
    want = np.flatnonzero(ok)[order]
    base = 64 + 2 * vocab
    assert np.array_equal(ints[base: base + n], want)
    assert np.array_equal(ints[base + batch * clen: base + batch * clen + n], k[want])
    count = np.bincount(k[ok], minlength=vocab)
    assert np.array_equal(info[:, 1], count) and np.array_equal(info[:, 0], np.cumsum(count) - count)

    got = gradient(hip, ix, dy, vocab, scale, acc, old, shift)
    total, size = np.zeros((vocab, dim)), np.zeros((vocab, dim))
    np.add.at(total, k[ok], dy.reshape(-1, dim)[ok].astype(np.float64))
    np.add.at(size, k[ok], np.abs(dy.reshape(-1, dim)[ok]).astype(np.float64))
    full = total * float(scale) + (old if acc else 0)
    # n - 1 sums, the scale and the last sum
    tol = F32 * ((count[:, None] + 1) * size * float(scale) + 2 * np.abs(old) * acc)
    assert (np.abs(got - full) <= tol).all()
    if acc:
        assert np.array_equal(got[count == 0], old[count == 0])
    else:
        assert (got[count == 0] == 0).all()
    assert np.array_equal(got, gradient(hip, ix, dy, vocab, scale, acc, old, shift))  # and again the same


def test_no_tokens(hip):
    table = np.ones((40, 8), np.float32)
    gt, ix = hip.Buffer.from_array(table), hip.Buffer(hip.lib().mle_embed_sorted_index_bytes(0, 4, 40))
    hip.call("mle_embed_scaled_fwd", None, None, gt.ptr, None, 0, 4, 4, 8, 40, 1.0, ix.ptr, ix.nbytes)
    hip.call("mle_embed_sorted_grad", None, gt.ptr, None, ix.ptr, ix.nbytes, 0, 4, 8, 40, 1.0, 1, None, 0)
    assert (gt.numpy() == 1).all()
    hip.call("mle_embed_sorted_grad", None, gt.ptr, None, ix.ptr, ix.nbytes, 0, 4, 8, 40, 1.0, 0, None, 0)
    assert (gt.numpy() == 0).all()


def test_lookup_without_index(hip):
    r = rng(3)
    table, keys = r.standard_normal((70, 36)).astype(np.float32), ids(r, "uniform", 3, 9, 9, 70)
    gt, gk, go = hip.Buffer.from_array(table), hip.Buffer.from_array(keys), hip.Buffer.empty((27, 36))
    hip.call("mle_embed_scaled_fwd", None, go.ptr, gt.ptr, gk.ptr, 3, 9, 9, 36, 70, 1.0, None, 0)
    assert np.array_equal(go.numpy(), table[keys.reshape(-1)])


def test_one_index_serves_two_gradients(hip):
    """Different widths and scales from one index."""
    r = rng(4)
    keys = ids(r, "frequent", 4, 200, 200, 500)
    _, ix = forward(hip, keys, r.standard_normal((500, 8)).astype(np.float32), 200, 1.0)
    for dim, scale in ((8, 2.0), (96, 0.5)):
        dy = r.standard_normal((4, 200, dim)).astype(np.float32)
        got = gradient(hip, ix, dy, 500, scale, 0, np.zeros((500, dim), np.float32))
        ref = np.zeros((500, dim))
        np.add.at(ref, keys.reshape(-1), dy.reshape(-1, dim).astype(np.float64) * scale)
        assert np.allclose(got, ref, rtol=1e-5, atol=1e-5)
