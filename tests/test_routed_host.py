"""Refusals of the routed-row entry points that need no GPU."""
import pytest
import torch

import swiftmoe_b200 as S
from swiftmoe_b200 import _lib as L
from swiftmoe_b200 import build
from swiftmoe_b200._lib import SwiftMoEError


@pytest.fixture(scope="module")
def lib():
    build.build()
    return L.load()


def test_cpu_tensors_are_refused():
    x = torch.randn(4, 16).bfloat16()
    idx = torch.zeros((4, 2), dtype=torch.int32)
    plan = dict(counts=idx[0], offsets=idx[0], slot_row=idx.view(-1), row_token=idx.view(-1), rows_cap=8, T=4, k=2)
    w = torch.randn(2, 8, 16).bfloat16()
    off = torch.tensor([0, 2, 4], dtype=torch.int32)
    for call in (lambda: S.sort_tokens(x, idx, 2), lambda: S.unsort_tokens(x, plan),
                 lambda: S.grouped_linear(x, w, off), lambda: S.grouped_linear(x, w, off, activation="swish")):
        with pytest.raises(SwiftMoEError):
            call()


BF, F32, P = 2, 0, 4096   # P: a non-null, aligned address that is never used


def test_sort_and_unsort_refusals(lib):
    sort = lambda **a: lib.smoe_sort_rows(*{**dict(x=P, dt=BF, sr=P, w=None, T=4, k=2, d=8, rt=None, off=P, E=2, cap=8,  # noqa: E731
                                                   rows=P, y=None, dw=None, st=None), **a}.values())
    for bad in (dict(dt=7), dict(T=-1), dict(k=0), dict(d=0), dict(E=0), dict(cap=-1), dict(x=None), dict(sr=None),
                dict(off=None), dict(rows=None), dict(dw=P, w=P), dict(dw=P, y=P)):
        assert sort(**bad) == -1, bad
    assert sort(k=33) == -4 and sort(cap=1 << 31) == -4
    assert sort(T=0, cap=0) == 0
    un = lambda **a: lib.smoe_unsort_rows(*{**dict(y=P, dt=BF, sr=P, w=None, T=4, k=2, d=8, cap=8, res=None, out=P, x=None,  # noqa: E731
                                                   dw=None, st=None), **a}.values())
    for bad in (dict(dt=7), dict(T=-1), dict(k=0), dict(d=0), dict(cap=-1), dict(y=None), dict(sr=None), dict(out=None),
                dict(dw=P, w=P), dict(dw=P, x=P)):
        assert un(**bad) == -1, bad
    assert un(k=33) == -4 and un(T=0) == 0


def test_sort_tokens_refusals(lib):
    st = lambda **a: lib.smoe_sort_tokens(*{**dict(x=P, dt=BF, idx=P, w=None, T=4, k=2, d=8, E=3, cap=0, al=1, cnt=P, off=P,  # noqa: E731
                                                   sr=P, rt=P, rows_cap=8, rows=P, ws=P, wsb=1 << 20, st=None), **a}.values())
    for bad in (dict(dt=7), dict(T=-1), dict(k=0), dict(d=0), dict(E=0), dict(al=0), dict(x=None), dict(idx=None),
                dict(cnt=None), dict(off=None), dict(sr=None), dict(rt=None), dict(rows=None), dict(rows_cap=7)):
        assert st(**bad) == -1, bad
    assert st(k=33) == -4 and st(ws=None) == -5 and st(wsb=8) == -5


def test_linear_refusals(lib):
    lin = lambda **a: lib.smoe_grouped_linear(*{**dict(A=P, W=P, lay=0, b=None, bdt=BF, act=0, res=None, z=None, fill=1, C=P,  # noqa: E731
                                                       dt=BF, off=P, G=2, R=300, N=16, K=16, ws=None, wsb=0, st=None), **a}.values())
    for bad in (dict(G=0), dict(N=0), dict(K=0), dict(R=-1), dict(act=5), dict(act=-1), dict(lay=2), dict(A=None),
                dict(W=None), dict(C=None), dict(off=None)):
        assert lin(**bad) == -1, bad
    for bad in (dict(dt=F32), dict(b=P, bdt=1), dict(N=12), dict(K=12), dict(G=1025), dict(R=1 << 31), dict(A=P + 2),
                dict(W=P + 8), dict(C=P + 4), dict(b=P + 2), dict(res=P + 2), dict(z=P + 2)):
        assert lin(**bad) == -4, bad
    assert lin(R=0) == 0
    act = lambda **a: lib.smoe_linear_act_bwd(*{**dict(dout=P, z=P, act=2, dz=P, db=None, bdt=BF, dt=BF, off=P, G=2, R=30, N=16,  # noqa: E731
                                                       ws=None, wsb=0, st=None), **a}.values())
    for bad in (dict(G=0), dict(N=0), dict(R=-1), dict(act=5), dict(dout=None), dict(z=None), dict(dz=None), dict(off=None)):
        assert act(**bad) == -1, bad
    for bad in (dict(dt=F32), dict(db=P, bdt=1), dict(N=12), dict(G=1025), dict(dout=P + 2), dict(z=P + 2), dict(dz=P + 2)):
        assert act(**bad) == -4, bad
    assert act(db=P) == -5 and act(R=0) == 0 and act(act=0) == 0
    wg = lambda **a: lib.smoe_linear_wgrad(*{**dict(dz=P, A=P, dt=BF, off=P, G=2, R=30, N=16, K=16, dW=P, odt=BF, ws=None, wsb=0, st=None),  # noqa: E731
                                             **a}.values())
    for bad in (dict(G=0), dict(N=0), dict(K=0), dict(R=-1), dict(dz=None), dict(A=None), dict(off=None), dict(dW=None)):
        assert wg(**bad) == -1, bad
    for bad in (dict(dt=F32), dict(odt=1), dict(N=12), dict(K=12), dict(G=1025), dict(dz=P + 2), dict(A=P + 2), dict(dW=P + 2)):
        assert wg(**bad) == -4, bad


def test_linear_backward_refusals(lib):
    bwd = lambda **a: lib.smoe_grouped_linear_bwd(*{**dict(dout=P, A=P, W=P, z=P, act=2, dt=BF, off=P, G=2, R=30, N=16, K=16,  # noqa: E731
                                                           dA=P, dW=P, db=P, bdt=BF, ws=P, wsb=1 << 26, st=None), **a}.values())
    for bad in (dict(G=0), dict(N=0), dict(K=0), dict(R=-1), dict(act=9), dict(dout=None), dict(z=None), dict(off=None)):
        assert bwd(**bad) == -1, bad
    for bad in (dict(dt=F32), dict(N=12), dict(bdt=1), dict(ws=P + 8), dict(dout=P + 2)):
        assert bwd(**bad) == -4, bad
    assert bwd(ws=None) == -5 and bwd(wsb=100) == -5
    size = lib.smoe_grouped_linear_bwd_workspace_size
    assert size(0, 7, BF, 0, 2, 16, 16) == 0 and size(0, 1, BF, 20000, 2, 16, 128) == 0
    assert size(2, 0, BF, 100, 2, 16, 16) == 3328                         # dz alone, 256-byte slabs
    assert size(2, 4, BF, 100, 2, 16, 16) > 3328


def test_workspace_sizes(lib):
    # partial tiles only where a launch can have few of them
    assert lib.smoe_grouped_linear_workspace_size(2, 4096, 4096, 8, L.SMOE_W_NK) == 0       # decode kernel
    assert lib.smoe_grouped_linear_workspace_size(2, 4096, 4096, 8, L.SMOE_W_KN) > 0
    assert 0 < lib.smoe_grouped_linear_workspace_size(64, 4096, 4096, 1, L.SMOE_W_NK) <= 64 << 20
    assert lib.smoe_grouped_linear_workspace_size(64, 4096, 128, 1, L.SMOE_W_NK) == 0       # short K
    assert lib.smoe_grouped_linear_workspace_size(16384, 4096, 4096, 8, L.SMOE_W_NK) == 0
    assert 0 < lib.smoe_linear_wgrad_workspace_size(32768, 1, 512, 512) <= 64 << 20
    assert lib.smoe_linear_wgrad_workspace_size(16384, 8, 14336, 4096) == 0
    # bias partials: a row per slice (16 to 512 rows) and one per group
    assert lib.smoe_linear_act_bwd_workspace_size(64, 8, 4) == (4 + 4) * 8 * 4
    assert lib.smoe_linear_act_bwd_workspace_size(1 << 20, 8, 4) == ((1 << 20) // 512 + 4) * 8 * 4


def test_largest_sizes(lib):
    # the last sizes the 32-bit counters of the kernels can pass are refused before any launch
    most, cols = (1 << 31) - 1 - 65535, (1 << 30) + 8
    assert lib.smoe_sort_rows(P, BF, P, None, 4, 2, 8, None, P, 2, most + 1, P, None, None, None) == -4
    assert lib.smoe_sort_rows(P, BF, P, None, 4, 2, cols, None, P, 2, 8, P, None, None, None) == -4
    assert lib.smoe_unsort_rows(P, BF, P, None, 4, 2, 8, most + 1, None, P, None, None, None) == -4
    assert lib.smoe_unsort_rows(P, BF, P, None, 4, 2, cols, 8, None, P, None, None, None) == -4
    for rows, n, k in ((most + 1, 8, 8), (8, cols, 8), (8, 8, cols)):
        assert lib.smoe_grouped_linear(P, P, 0, None, BF, 0, None, None, 1, P, BF, P, 2, rows, n, k, None, 0, None) == -4
        assert lib.smoe_linear_wgrad(P, P, BF, P, 2, rows, n, k, P, BF, None, 0, None) == -4
    for rows, n in ((most + 1, 8), (8, cols)):
        assert lib.smoe_linear_act_bwd(P, P, 2, P, None, BF, BF, P, 2, rows, n, None, 0, None) == -4
    # the bias gradient's slices of rows are a grid's y blocks
    for rows in (512 * 65535, 512 * 65535 + 1, 1 << 26, most):
        for n in (8, 64, 4096):
            slices = lib.smoe_linear_act_bwd_workspace_size(rows, n, 4) // (n * 4) - 4
            assert 0 < slices <= 65535, (rows, n, slices)
