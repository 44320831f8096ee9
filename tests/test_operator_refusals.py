"""What the vocabulary cross entropy, the 8-bit checkpoints, the norm with 8-bit
output and the sorted embedding refuse: before anything is launched, so this
runs without a GPU.  Pointers are made up; none is followed."""
import re

import pytest

from ml_engine_amd import hip

A = 1 << 20  # an aligned address
BIG = (1 << 30) + 1


def refused(match, name, *args):
    rc = getattr(hip.lib(), name)(*args)
    assert rc in (-1, -4, -5), (name, rc)  # argument, unsupported size, workspace
    message = hip.lib().mle_last_error().decode()
    assert re.search(match, message), message


# the calls' arguments in order, each a right call on rows x cols data
XENT_FWD = dict(stream=None, rows=8, d=16, vocab=32, X=A, ldx=16, W=A, ldw=32, bias=A, keys=A, clen=8, max_clen=8,
                loss_scale=1.0, lse=A, row_loss=A, loss=A, ws=A, ws_bytes=1 << 40)
XENT_BWD = dict(stream=None, rows=8, d=16, vocab=32, X=A, ldx=16, W=A, ldw=32, bias=A, keys=A, clen=8, max_clen=8, lse=A,
                upstream=None, grad_scale=1.0, dX=A, lddx=16, acc_dx=0, dW=A, lddw=32, db=A, acc_dw=0, ws=A,
                ws_bytes=1 << 40)
QUANT = dict(stream=None, rows=8, cols=40, x=A, ldx=40, q=A, ldq=40, e=A, lde=2)
DEQUANT = dict(stream=None, rows=8, cols=40, q=A, ldq=40, e=A, lde=2, y=A, ldy=40)
ACT_FWD = dict(stream=None, kind=1, rows=8, cols=40, x=A, ldx=40, y=A, ldy=40, q=A, ldq=40, e=A, lde=2)
ACT_BWD = dict(stream=None, kind=1, rows=8, cols=40, q=A, ldq=40, e=A, lde=2, dy=A, lddy=40, dx=A, lddx=40, acc=0)
WGRAD = dict(stream=None, rows=4096, inp=40, out=24, q=A, ldq=40, e=A, lde=2, dY=A, lddy=24, dW=A, lddw=24, db=A, acc=0, ws=A,
             ws_bytes=1 << 40)
NORM_FWD = dict(stream=None, rows=8, cols=40, x=A, r=A, w=A, eps=1e-5, h=A, y=A, rstd=A, q=A, ldq=40, e=A, lde=2)
NORM_BWD = dict(stream=None, rows=8, cols=40, h=A, w=A, rstd=A, dy=A, dres=A, dh=A, acc_dh=0, dw=A, acc_dw=0, ws=A,
                ws_bytes=1 << 40)
EMBED_FWD = dict(stream=None, out=A, table=A, keys=A, batch=2, clen=4, max_clen=4, dim=16, vocab=32, scale=1.0, index=A,
                 index_bytes=1 << 40)
EMBED_BWD = dict(stream=None, dtable=A, dy=A, index=A, index_bytes=1 << 40, batch=2, clen=4, dim=16, vocab=32, scale=1.0,
                 acc=0, ws=A, ws_bytes=1 << 40)

CASES = [
    ("mle_vocab_xent_fwd", XENT_FWD, [dict(rows=-1), dict(d=0), dict(vocab=0), dict(X=None), dict(W=None), dict(keys=None),
                                      dict(ldx=15), dict(ldw=31), dict(clen=0), dict(max_clen=7), dict(lse=None),
                                      dict(loss=None), dict(ws=None), dict(ws=A + 4), dict(ws_bytes=64),
                                      dict(rows=BIG), dict(d=BIG, ldx=BIG), dict(vocab=BIG, ldw=BIG)]),
    ("mle_vocab_xent_bwd", XENT_BWD, [dict(rows=-1), dict(X=None), dict(W=None), dict(keys=None), dict(lse=None),
                                      dict(lddx=15), dict(lddw=31), dict(dW=None), dict(ws=None), dict(ws=A + 8),
                                      dict(ws_bytes=64), dict(max_clen=7), dict(rows=BIG), dict(d=BIG, ldx=BIG, lddx=BIG),
                                      dict(vocab=BIG, ldw=BIG, lddw=BIG)]),
    ("mle_q8_quantize", QUANT, [dict(rows=-1), dict(cols=0), dict(x=None), dict(q=None), dict(e=None), dict(ldx=39),
                                dict(ldq=39), dict(lde=1), dict(cols=BIG, ldx=BIG, ldq=BIG, lde=BIG)]),
    ("mle_q8_dequantize", DEQUANT, [dict(rows=-1), dict(cols=-3), dict(y=None), dict(q=None), dict(e=None), dict(ldy=39),
                                    dict(ldq=39), dict(lde=1)]),
    ("mle_q8_act_fwd", ACT_FWD, [dict(kind=-1), dict(kind=6), dict(x=None), dict(y=None), dict(q=None), dict(ldx=39),
                                 dict(ldy=39), dict(lde=1)]),
    ("mle_q8_act_bwd", ACT_BWD, [dict(kind=-1), dict(kind=6), dict(dy=None), dict(dx=None), dict(e=None), dict(lddy=39),
                                 dict(lddx=39), dict(ldq=39)]),
    ("mle_q8_linear_wgrad", WGRAD, [dict(rows=-1), dict(inp=0), dict(out=0), dict(q=None), dict(e=None), dict(dY=None),
                                    dict(dW=None), dict(ldq=39), dict(lde=1), dict(lddy=23), dict(lddw=23), dict(ws=None),
                                    dict(ws=A + 4), dict(ws_bytes=64), dict(rows=BIG),
                                    dict(inp=BIG, ldq=BIG, lde=BIG), dict(out=BIG, lddw=BIG), dict(lddy=1 << 24)]),
    ("mle_add_rmsnorm_q8_fwd", NORM_FWD, [dict(rows=-1), dict(cols=0), dict(x=None), dict(rstd=None), dict(q=None),
                                          dict(e=None), dict(ldq=39), dict(lde=1), dict(eps=-1.0),
                                          dict(eps=float("nan")), dict(cols=BIG, ldq=BIG, lde=BIG)]),
    ("mle_add_rmsnorm_bwd", NORM_BWD, [dict(rows=-1), dict(cols=0), dict(h=None), dict(rstd=None), dict(dy=None),
                                       dict(dh=None), dict(ws=None), dict(ws=A + 4), dict(ws_bytes=64), dict(cols=BIG)]),
    ("mle_embed_scaled_fwd", EMBED_FWD, [dict(batch=-1), dict(clen=0), dict(max_clen=3), dict(dim=0), dict(vocab=0),
                                         dict(out=None), dict(table=None), dict(keys=None), dict(index=A + 4),
                                         dict(index_bytes=64), dict(batch=1 << 20, clen=1 << 11, max_clen=1 << 11),
                                         dict(dim=BIG), dict(vocab=BIG)]),
    ("mle_embed_sorted_grad", EMBED_BWD, [dict(batch=-1), dict(clen=0), dict(dim=0), dict(vocab=0), dict(dtable=None),
                                          dict(dy=None), dict(index=None), dict(index=A + 4), dict(index_bytes=64),
                                          dict(ws=None), dict(ws=A + 8), dict(ws_bytes=64),
                                          dict(batch=1 << 20, clen=1 << 11), dict(batch=1 << 20, clen=64),
                                          dict(vocab=1 << 30), dict(dim=BIG), dict(vocab=BIG)]),
]


@pytest.mark.parametrize("name,right,wrong", [(n, r, w) for n, r, ws in CASES for w in ws],
                         ids=[f"{n}-{'-'.join(w)}-{i}" for n, r, ws in CASES for i, w in enumerate(ws)])
def test_refused(name, right, wrong):
    refused(name, name, *dict(right, **wrong).values())


@pytest.mark.parametrize("query", ["mle_vocab_xent_ws_bytes", "mle_q8_linear_wgrad_ws_bytes", "mle_embed_sorted_grad_ws_bytes"])
def test_queries_take_zeros(query):
    for zero in range(3):
        sizes = [64, 48, 40]
        sizes[zero] = 0
        assert getattr(hip.lib(), query)(*sizes) == 0
    assert getattr(hip.lib(), query)(64, 48, 40) > 0


def test_other_queries_take_zeros():
    L = hip.lib()
    assert L.mle_add_rmsnorm_ws_bytes(0, 40) == 0 == L.mle_add_rmsnorm_ws_bytes(40, 0)
    assert L.mle_embed_sorted_index_bytes(0, 4, 10) > 0  # the table's rows are listed with no tokens
    assert L.mle_embed_sorted_index_bytes(2, 0, 10) == 0 == L.mle_embed_sorted_index_bytes(2, 4, 0)


@pytest.mark.parametrize("rows,d,vocab", [(8192, 512, 8000), (8192, 1024, 32000), (16384, 4096, 128000), (65536, 1024, 50257)])
def test_vocab_xent_workspace_stays_below_the_logits(rows, d, vocab):
    """The workspace of large problems is a fraction of the logits and their
    gradient, which it replaces, beside what the weights and inputs take anyway."""
    need = hip.lib().mle_vocab_xent_ws_bytes(rows, d, vocab)
    assert need <= 0.6 * 8 * rows * vocab + 3 * 4 * (rows * d + d * vocab), need


@pytest.mark.parametrize("rows,d,vocab", [(1000, 330, 10007), (2048, 1024, 16000), (200, 1024, 32000), (300, 4096, 128000),
                                          (512, 1024, 4096), (192, 64, 16000), (4096, 512, 8000), (8192, 256, 1000),
                                          (200000, 16, 1100), (1000, 5000, 1000)])
def test_vocab_xent_workspace_of_middle_sizes(rows, d, vocab):
    """Where the logits themselves are no more than the workspace: 8 bytes for each logit of a
    piece (256 MiB at most), each element of X and of the piece's columns of W, in whole
    tiles of 128, and as much again for partial sums and statistics at most."""
    up = lambda n: -(-n // 128) * 128  # noqa: E731
    r, f = up(min(rows, 32768)), up(d)
    pieces = -(-vocab // max(128, (1 << 25) // r // 128 * 128))
    piece = up(-(-vocab // pieces))
    need = hip.lib().mle_vocab_xent_ws_bytes(rows, d, vocab)
    assert 0 < need <= 2 * 8 * (r * piece + f * (r + piece)), need
