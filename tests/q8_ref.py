"""The 8-bit format of kept activations, in numpy: every step is exact."""
import numpy as np

GROUP = 32


def quantize(x):
    """(codes int8 [rows, cols], exponent bytes [rows, groups]) of float32 x."""
    rows, cols = x.shape
    ng = -(-cols // GROUP)
    v = np.zeros((rows, ng * GROUP))
    v[:, :cols] = x
    v = v.reshape(rows, ng, GROUP)
    bad = ~np.isfinite(v).all(axis=2)
    top = np.abs(np.where(np.isfinite(v), v, 0)).max(axis=2)
    m, k = np.frexp(top)  # top = m 2^k, 1/2 <= m < 1
    k = np.clip(k - np.where(m < 127.5 / 128, 7, 6), -126, 121)
    k = np.where(top == 0, -126, k)
    with np.errstate(invalid="ignore", over="ignore"):
        q = np.clip(np.rint(np.ldexp(v, -k[:, :, None])), -127, 127)
    q = np.where(bad[:, :, None], np.where(np.isinf(v), np.sign(v), 0), q)
    e = np.where(bad, 255, k + 127).astype(np.uint8)
    return q.reshape(rows, -1)[:, :cols].astype(np.int8), e


def values(q, e):
    """float32 values of codes and exponent bytes."""
    step = (np.repeat(e.astype(np.uint32), GROUP, axis=1)[:, : q.shape[1]] << 23).view(np.float32)
    with np.errstate(invalid="ignore"):
        return q.astype(np.float32) * step


def kept(x):
    return values(*quantize(x))
