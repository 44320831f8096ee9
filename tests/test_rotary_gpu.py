"""Rotary positions of several axes against 64 bits."""
import ctypes as C
import math

import numpy as np
import pytest

from conftest import rng

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -24  # half a step of fp32
NEIGHBOURS, BY_AXIS = 1, 2


def turned(x, positions, sections, base, flags, inverse):
    """x [rows, heads, dim] in 64 bits."""
    n = sum(sections)
    axis = np.repeat(np.arange(len(sections)), sections)
    if flags & BY_AXIS:
        power = np.concatenate([np.arange(s) / max(s, 1) for s in sections])
    else:
        power = np.arange(n) / n
    angle = positions[axis].T.astype(np.float64) * base ** -power
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None] * (-1 if inverse else 1)
    y = x.astype(np.float64).copy()
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if flags & NEIGHBOURS else (slice(0, n), slice(n, 2 * n))
    u, v = y[:, :, a].copy(), y[:, :, b].copy()
    y[:, :, a], y[:, :, b] = u * c - v * s, u * s + v * c
    size = np.abs(y)
    size[:, :, a] = size[:, :, b] = np.abs(u) + np.abs(v)
    return y, size


def run(hip, x, y, positions, sections, base, flags, inverse, acc, ld):
    """x and y: [(device pointer, heads)] of q and k."""
    sec = (C.c_int * len(sections))(*sections)
    rows, dim = positions.shape[1], run.dim
    g = hip.Buffer.from_array(positions.astype(np.int32))
    hip.call("mle_rotary", None, rows, dim, x[0][0], ld, y[0][0], ld, x[0][1], x[1][0], ld, y[1][0], ld, x[1][1], g.ptr,
             len(sections), sec, base, flags, inverse, acc)
    hip.sync()


CASES = [  # rows heads kv dim sections far
    (1, 1, 0, 2, [1], 10), (3, 2, 1, 16, [8], 100), (5, 8, 8, 64, [16, 16], 300), (7, 16, 4, 128, [16, 24, 24], 10 ** 6),
    (33, 3, 1, 80, [10, 15, 15], 4000), (9, 4, 2, 72, [20], 50000), (4, 5, 5, 20, [1, 0, 6], 900), (2, 2, 1, 256, [128], 2 ** 20),
    (130, 6, 2, 40, [3, 5, 7], 10 ** 5), (3000, 2, 1, 64, [32], 3000), (2, 3, 2, 254, [127], 77), (11, 1, 1, 33, [4, 4, 4, 4], 50),
    (6, 40, 3, 24, [12], 9), (2, 1, 1, 64, [1, 2, 3, 4, 5, 6, 7, 4], 1000),
]


@pytest.mark.parametrize("rows,heads,kv,dim,sections,far", CASES)
@pytest.mark.parametrize("flags,inverse,acc,pad,shift", [(0, 0, 0, 0, 0), (1, 1, 0, 0, 0), (2, 0, 1, 5, 1), (3, 1, 1, 3, 3), (0, 1, 1, 4, 0), (1, 0, 0, 1, 2)])
def test_against_64_bits(hip, rows, heads, kv, dim, sections, far, flags, inverse, acc, pad, shift):
    r = rng(rows + dim)
    ld = max(heads, kv) * dim + pad
    pos = r.integers(-far, far + 1, (len(sections), rows)).astype(np.int32)
    run.dim = dim
    bufs, host, old = [], [], []
    for h in (heads, kv):
        x, o = (r.standard_normal((rows, ld)).astype(np.float32) for _ in range(2))
        host.append(x)
        old.append(o)
        bufs.append([hip.Buffer.from_array(np.concatenate([np.zeros(shift, np.float32), a.reshape(-1)])) for a in (x, o)])
    at = lambda b: b.ptr + 4 * shift  # noqa: E731
    run(hip, [(at(bufs[0][0]), heads), (at(bufs[1][0]), kv)], [(at(bufs[0][1]), heads), (at(bufs[1][1]), kv)], pos, sections, 10000.0,
        flags, inverse, acc, ld)
    for i, h in enumerate((heads, kv)):
        got = bufs[i][1].numpy()[shift:].reshape(rows, ld)
        assert np.array_equal(got[:, h * dim:], old[i][:, h * dim:])  # beside the heads nothing is written
        if h == 0:
            continue
        want, size = turned(host[i][:, :h * dim].reshape(rows, h, dim), pos, sections, 10000.0, flags, inverse)
        tol = size.copy()
        if acc:
            o = old[i][:, :h * dim].reshape(rows, h, dim)
            want, tol = want + o, size + 0.5 * (np.abs(o) + size)
        # cos and sin, two products, a sum (and the sum with what was there) round; the angle's own last
        # place in 64 bits, a frequency's rounding times a position, is 2^-52 of it at most twice
        assert (np.abs(got[:, :h * dim].reshape(rows, h, dim) - want) <= (4 * F32 + 2.0 ** -50 * far) * tol).all()


def test_in_place_and_back(hip):
    """In place gives the same bits, and the inverse turn brings the values back."""
    r = rng(4)
    rows, heads, kv, dim, sections = 50, 6, 2, 96, [16, 16, 16]
    run.dim = dim
    ld = heads * dim
    pos = r.integers(0, 10 ** 6, (3, rows)).astype(np.int32)
    q, k = (r.standard_normal((rows, ld)).astype(np.float32) for _ in range(2))
    for flags in range(4):
        gq, gk, oq, ok = (hip.Buffer.from_array(a) for a in (q, k, q, k))
        run(hip, [(gq.ptr, heads), (gk.ptr, kv)], [(oq.ptr, heads), (ok.ptr, kv)], pos, sections, 5e5, flags, 0, 0, ld)
        run(hip, [(gq.ptr, heads), (gk.ptr, kv)], [(gq.ptr, heads), (gk.ptr, kv)], pos, sections, 5e5, flags, 0, 0, ld)
        assert np.array_equal(gq.numpy(), oq.numpy()) and np.array_equal(gk.numpy(), ok.numpy())
        run(hip, [(gq.ptr, heads), (gk.ptr, kv)], [(gq.ptr, heads), (gk.ptr, kv)], pos, sections, 5e5, flags, 1, 0, ld)
        # there and back: each way off by at most 4 roundings of |a| + |b| <= 2 max
        assert np.abs(gq.numpy() - q).max() <= 16 * F32 * 2 * np.abs(q).max()
        assert np.array_equal(gk.numpy()[:, kv * dim:], k[:, kv * dim:])


def test_far_positions(hip):
    """The largest int32 positions: a frequency of 1 is exact, so the angle is good to its last place in 64 bits."""
    pos = np.array([[2 ** 31 - 1, -2 ** 31, 123456789, 0]], np.int32)
    x = np.ones((4, 2), np.float32)
    x[:, 1] = 0
    g = hip.Buffer.from_array(x)
    run.dim = 2
    run(hip, [(g.ptr, 1), (None, 0)], [(g.ptr, 1), (None, 0)], pos, [1], 10000.0, 0, 0, 0, 2)
    got = g.numpy()
    for i, p in enumerate(pos[0]):
        # the kernel's turns are p / 2 pi in 64 bits: two roundings of 2^-53 of up to 2^31 / 2 pi turns
        tol = 2 * F32 + 2 * 2.0 ** -53 * abs(int(p)) * 2
        assert abs(got[i, 0] - math.cos(int(p))) <= tol and abs(got[i, 1] - math.sin(int(p))) <= tol
    assert got[3, 0] == 1 and got[3, 1] == 0


def test_not_finite(hip):
    """A value that is not finite reaches its pair alone."""
    x = rng(5).standard_normal((6, 64)).astype(np.float32)
    x[2, 7], x[4, 40] = np.nan, np.inf
    g, o = hip.Buffer.from_array(x), hip.Buffer.empty((6, 64))
    run.dim = 64
    run(hip, [(g.ptr, 1), (None, 0)], [(o.ptr, 1), (None, 0)], np.arange(1, 7, dtype=np.int32)[None], [32], 1e4, 0, 0, 0, 64)
    bad = ~np.isfinite(o.numpy())
    assert sorted(map(tuple, np.argwhere(bad))) == [(2, 7), (2, 39), (4, 8), (4, 40)]


def test_no_rows(hip):
    sec = (C.c_int * 1)(8)
    hip.call("mle_rotary", None, 0, 16, None, 16, None, 16, 1, None, 0, None, 0, 0, None, 1, sec, 1e4, 0, 0, 0)
