"""What windowed attention, the rotary positions and the layer norm with a weight
refuse: before anything is launched, so this runs without a GPU.  Pointers are made
up; none is followed."""
import ctypes as C

import pytest

from ml_engine_amd import hip
from test_operator_refusals import A, BIG, refused

SEC = (C.c_int * 3)(4, 6, 6)
NEG = (C.c_int * 3)(4, -1, 6)
NONE = (C.c_int * 3)(0, 0, 0)

FWD = dict(stream=None, q=A, ldq=256, k=A, ldk=128, v=A, ldv=128, out=A, ldo=256, lse=A, lengths=A, batch=2, seq=40, heads=4,
           kv_heads=2, dim=64, scale=0.125, window=16, sinks=2)
BWD = dict(stream=None, q=A, ldq=256, k=A, ldk=128, v=A, ldv=128, out=A, ldo=256, lse=A, dout=A, lddo=256, dq=A, lddq=256,
           acc_q=0, dk=A, lddk=128, acc_k=0, dv=A, lddv=128, acc_v=0, lengths=A, batch=2, seq=40, heads=4, kv_heads=2, dim=64,
           scale=0.125, window=16, sinks=2, ws=A, ws_bytes=1 << 40)
STEP = dict(stream=None, q=A, ldq=256, k=A, ldk=128, v=A, ldv=128, out=A, ldo=256, lengths=A, batch=2, tokens=1, capacity=4000,
            heads=4, kv_heads=2, dim=64, scale=0.125, window=3000, sinks=2, ws=A, ws_bytes=1 << 40)
ROTARY = dict(stream=None, rows=8, dim=40, q=A, ldq=160, q_out=A, ldqo=160, heads=4, k=A, ldk=80, k_out=A, ldko=80, kv_heads=2,
              positions=A, axes=3, sections=SEC, base=1e4, flags=0, inverse=0, acc=0)
LN_FWD = dict(stream=None, rows=8, cols=40, x=A, r=A, w=A, b=A, eps=1e-5, h=A, y=A, mean=A, rstd=A)
LN_BWD = dict(stream=None, rows=8, cols=40, h=A, w=A, mean=A, rstd=A, dy=A, dres=A, dh=A, acc_dh=0, dw=A, db=A, acc_dw=0, ws=A,
              ws_bytes=1 << 40)

SHAPE = [dict(heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(dim=0), dict(dim=129, ldq=1000, ldk=1000, ldv=1000, ldo=1000),
         dict(scale=float("nan")), dict(scale=float("inf")), dict(window=0), dict(window=-5), dict(sinks=-1), dict(ldq=255),
         dict(ldk=127), dict(ldv=127), dict(ldo=255), dict(batch=-1), dict(q=None), dict(k=None), dict(v=None), dict(out=None),
         dict(batch=BIG), dict(batch=1 << 24, heads=1 << 16, kv_heads=1 << 16, dim=1, ldq=1 << 16, ldk=1 << 16, ldv=1 << 16, ldo=1 << 16)]
CASES = [
    ("mle_window_attention_fwd", FWD, SHAPE + [dict(seq=-1), dict(seq=BIG)]),
    ("mle_window_attention_bwd", BWD, SHAPE[:-1] + [dict(seq=-1), dict(seq=BIG), dict(lse=None), dict(dout=None), dict(dq=None),
                                                    dict(dk=None), dict(dv=None), dict(lddo=255), dict(lddq=255),
                                                    dict(lddk=127), dict(lddv=127), dict(ws=None), dict(ws=A + 4),
                                                    dict(ws_bytes=64)]),
    ("mle_window_attention_step", STEP, SHAPE + [dict(tokens=-1), dict(tokens=BIG), dict(capacity=-1), dict(capacity=BIG),
                                                 dict(lengths=None), dict(ws=None), dict(ws=A + 8), dict(ws_bytes=64)]),
    ("mle_rotary", ROTARY, [dict(rows=-1), dict(dim=0), dict(dim=31), dict(heads=0), dict(kv_heads=-1), dict(q=None),
                            dict(q_out=None), dict(k=None), dict(k_out=None), dict(positions=None), dict(ldq=159),
                            dict(ldqo=159), dict(ldk=79), dict(ldko=79), dict(axes=0), dict(axes=9), dict(sections=None),
                            dict(sections=NEG), dict(sections=NONE), dict(base=0.0), dict(base=-1.0),
                            dict(base=float("nan")), dict(base=float("inf")), dict(flags=4), dict(flags=-1),
                            dict(dim=300, ldq=1200, ldqo=1200, ldk=600, ldko=600, sections=(C.c_int * 3)(100, 20, 20))]),
    ("mle_add_layernorm_fwd", LN_FWD, [dict(rows=-1), dict(cols=0), dict(cols=BIG), dict(x=None), dict(mean=None),
                                       dict(rstd=None), dict(eps=-1.0), dict(eps=float("nan"))]),
    ("mle_add_layernorm_bwd", LN_BWD, [dict(rows=-1), dict(cols=0), dict(cols=BIG), dict(h=None), dict(mean=None),
                                       dict(rstd=None), dict(dy=None), dict(dh=None), dict(ws=None), dict(ws=A + 4),
                                       dict(ws_bytes=64), dict(dw=None, ws=None), dict(db=None, ws_bytes=16)]),
]


@pytest.mark.parametrize("name,right,wrong", [(n, r, w) for n, r, ws in CASES for w in ws],
                         ids=[f"{n}-{'-'.join(w)}-{i}" for n, r, ws in CASES for i, w in enumerate(ws)])
def test_refused(name, right, wrong):
    refused(name, name, *dict(right, **wrong).values())


def test_queries_take_zeros():
    L = hip.lib()
    right = [2, 40, 4, 2, 64, 16, 2]
    assert L.mle_window_attention_ws_bytes(*right) > 0
    for i in range(5):
        assert L.mle_window_attention_ws_bytes(*(right[:i] + [0] + right[i + 1:])) == 0
    right = [2, 1, 4000, 4, 2, 64, 3000, 2]
    assert L.mle_window_attention_step_ws_bytes(*right) > 0
    for i in range(6):
        assert L.mle_window_attention_step_ws_bytes(*(right[:i] + [0] + right[i + 1:])) == 0
    assert L.mle_add_layernorm_ws_bytes(0, 40) == 0 == L.mle_add_layernorm_ws_bytes(40, 0)


def test_workspace_of_many_sinks():
    """The far parts of sinks take no more than some tensors of the keys' size."""
    lib = hip.lib()
    for batch, seq, kv, dim in ((1, 8192, 8, 128), (8, 8192, 8, 128), (1, 100000, 1, 64), (64, 4096, 4, 64)):
        for sinks in (1, 1000, seq // 2, seq):
            tensor = 4 * batch * seq * kv * dim
            assert lib.mle_window_attention_ws_bytes(batch, seq, kv, kv, dim, 1, sinks) <= (1 << 29) + 4 * tensor


def test_workspaces_stay_small():
    """The backward's is a number per row and head and a share of the sinks' gradients; a step's, partial rows."""
    L = hip.lib()
    assert L.mle_window_attention_ws_bytes(2, 4096, 16, 4, 128, 1024, 4) <= 16 << 20
    assert L.mle_window_attention_step_ws_bytes(32, 1, 8192, 32, 8, 128, 4096, 4) <= 32 << 20
