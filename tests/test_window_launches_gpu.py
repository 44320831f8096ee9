"""Windowed attention in each form that its launches choose from: the forward's waves to a
workgroup and to 32 rows, workgroups numbered by group of heads or by their place in it, groups
that fill the 8 XCDs evenly or not, keys' sums whole or in parts, sinks' far rows, at each width.
Some groups of heads against 64 bits, the others for having been written."""
import numpy as np
import pytest

import wattn_ref as ref
from conftest import rng
from test_window_attention_gpu import Case, Step

pytestmark = pytest.mark.gpu

# batch, seq, heads, heads of keys, window, sinks, some lengths, accumulated gradients
FORMS = {
    # forward with 8 waves to 256 rows (windows of 512 and more)
    "rows of 8 waves, by group": (8, 520, 16, 4, 513, 4, 1, 7),
    "rows of 8 waves, by group, groups not in eights": (15, 515, 12, 3, 600, 2, 0, 0),
    "rows of 8 waves, by place": (12, 520, 8, 8, 512, 0, 1, 2),
    # two waves to 32 rows, 64 and 128 rows to a workgroup
    "64 rows, by group": (4, 500, 4, 2, 90, 3, 1, 5),
    "128 rows of pairs, by group": (4, 500, 16, 4, 150, 0, 0, 0),
    # 4 waves to 128 rows; whole sums of keys, and the sinks' far rows added to them
    "rows of 4 waves, by group; whole near sums and far ones": (8, 500, 16, 4, 100, 4, 1, 7),
    "rows of 4 waves, by group, not in eights; far sums": (15, 500, 12, 3, 100, 200, 0, 7),
    # more workgroups of the backward than are numbered by place
    "backward by group": (17, 400, 16, 16, 64, 3, 1, 7),
    "backward by group, groups not in eights": (13, 500, 11, 11, 64, 3, 0, 2),
}


@pytest.mark.parametrize("dim", [64, 40, 80, 96, 128, 121])
@pytest.mark.parametrize("form", FORMS)
def test_forms(hip, form, dim):
    b, n, h, kv, w, s, lengths, acc = FORMS[form]
    r = rng(dim + n)
    lengths = np.where(r.random(b) < 0.3, r.integers(0, n + 1, b), n) if lengths else None
    c = Case(hip, b, n, h, kv, dim, w, s, lengths, acc=acc)
    c.forward()
    c.backward()
    got, g = c.results(), h // kv
    for name, a in got.items():
        assert not np.isnan(a).any(), name
    pick = {(0, 0), (b - 1, kv - 1)} | {(int(r.integers(b)), int(r.integers(kv))) for _ in range(2)}
    for i, e in sorted(pick):
        q, k = slice(e * g, (e + 1) * g), slice(e, e + 1)
        t = ref.whole(c.q[i:i + 1, :, q], c.k[i:i + 1, :, k], c.v[i:i + 1, :, k], None if lengths is None else lengths[i:i + 1], g, 1,
                      w, s, c.scale, c.dout[i:i + 1, :, q])
        for j, (name, at) in enumerate((("dq", q), ("dk", k), ("dv", k))):
            ref.check(got[name][i:i + 1, :, at], t, name, c.old[j][i:i + 1, :, at] if acc >> j & 1 else None)
        ref.check(got["out"][i:i + 1, :, q], t, "out")
        ref.check(got["lse"][i:i + 1, q], t, "lse")


# batch, capacity, heads, heads of keys, dim, window, sinks, equal lengths
STEPS = [
    (33, 2700, 8, 8, 32, 9000, 0, 0),   # unlike lengths over whole caches: keys in parts
    (26, 5200, 32, 8, 16, 5200, 0, 0),
    (33, 1300, 8, 8, 48, 1100, 4, 1),   # a few groups past a round of the CUs
    (66, 1700, 16, 8, 32, 1600, 0, 0),
    (32, 1400, 8, 8, 64, 1100, 4, 0),   # whole groups
    (30, 700, 8, 8, 40, 700, 0, 0),
]


@pytest.mark.parametrize("b,cap,h,kv,dim,w,s,equal", STEPS)
def test_steps_of_many_groups(hip, b, cap, h, kv, dim, w, s, equal):
    r = rng(cap)
    lengths = np.full(b, cap) if equal else r.integers(0, cap + 1, b)
    t = Step(hip, b, 1, cap, h, kv, dim, w, s, lengths)
    t.run()
    t.check()
    one = t.out.get()
    t.run()
    assert np.array_equal(one, t.out.get())
