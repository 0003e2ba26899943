"""The operators for vocabularies refuse bad arguments before they touch a GPU, and say how much scratch they need."""
import ctypes as C

import pytest

from lbtree import _lib

L = _lib.lib
# addresses far apart, never followed: the checks come first
AT, W, Y, OUT, GX, GW, GB, WS = (C.c_void_p((i + 1) << 50) for i in range(8))
ODD = C.c_void_p((9 << 50) + 8)
BIG = 1 << 40


def loss(stream=None, X=AT, weight=W, dtype=_lib.LBT_BF16, n=10, f=8, k=100, bias=None, y=Y, out=OUT, ws=None, size=0):
    return L.lbt_linear_log_loss(stream, X, weight, dtype, n, f, k, bias, y, out, ws, size)


def gradient(X=AT, weight=W, dtype=_lib.LBT_BF16, n=10, f=8, k=100, bias=None, y=Y, w=None, out=OUT, gx=GX, gw=GW, gb=None,
             ws=None, size=0):
    return L.lbt_linear_log_loss_gradient(None, X, weight, dtype, n, f, k, bias, y, w, out, gx, gw, gb, ws, size)


@pytest.mark.parametrize("arguments,message", [
    (dict(dtype=_lib.LBT_F64), b"dtype"), (dict(dtype=9), b"dtype"), (dict(dtype=-1), b"dtype"),
    (dict(n=-1), b"shape"), (dict(f=0), b"shape"), (dict(k=0), b"shape"), (dict(k=-5), b"shape"),
    (dict(n=1 << 31), b"shape"), (dict(f=1 << 20, k=1 << 20), b"shape"),
    (dict(X=None), b"null"), (dict(weight=None), b"null"), (dict(y=None), b"null"), (dict(out=None), b"null"),
    (dict(X=ODD), b"aligned"), (dict(weight=ODD), b"aligned"),
])
def test_loss_refuses(arguments, message):
    for call in (loss, gradient):
        assert call(**arguments) == -1
        assert message in L.lbt_last_error()


@pytest.mark.parametrize("arguments,message", [
    (dict(gx=None), b"null"), (dict(gw=None), b"null"), (dict(gx=ODD), b"aligned"), (dict(gw=ODD), b"aligned"),
    (dict(gb=GB), b"without a bias"),
])
def test_gradient_refuses(arguments, message):
    assert gradient(**arguments) == -1
    assert message in L.lbt_last_error()


def test_workspaces_are_checked():
    for call, grad in ((loss, 0), (gradient, 1)):
        need = L.lbt_linear_log_loss_workspace_bytes(10, 8, 100, _lib.LBT_BF16, grad)
        assert need > 0
        assert call(ws=None) == -3 and b"workspace" in L.lbt_last_error()
        assert call(ws=WS, size=need - 1) == -3 and str(need).encode() in L.lbt_last_error()
        assert call(ws=ODD, size=BIG) == -3 and b"aligned" in L.lbt_last_error()


def test_workspace_sizes():
    q = L.lbt_linear_log_loss_workspace_bytes
    assert q(10, 8, 100, _lib.LBT_F64, 0) == 0 and q(-1, 8, 100, _lib.LBT_BF16, 0) == 0 and q(10, 0, 100, _lib.LBT_BF16, 1) == 0
    assert q(0, 8, 100, _lib.LBT_BF16, 1) > 0
    for dtype in (_lib.LBT_BF16, _lib.LBT_F16, _lib.LBT_F32):
        assert q(1000, 64, 5000, dtype, 0) <= q(1000, 64, 5000, dtype, 1)
        assert q(1000, 64, 5000, dtype, 1) < q(1000, 64, 5000, dtype, 2)
        assert q(1000, 64, 5000, dtype, 3) == 0 and q(1000, 64, 5000, dtype, -1) == 0
        # a piece of the gradient takes 4 GiB at most and one of packed weights 512 MiB, whatever the vocabulary: the rest is the
        # shares of the rows' totals, 2 x 8 bytes a row and 256 classes, and what is as large as X
        assert q(8192, 4096, 1 << 20, dtype, 1) < (7 << 30)
    # the scores of 8192 rows and a million classes would take 32 GiB
    assert q(8192, 1024, 1 << 20, _lib.LBT_BF16, 0) < (1 << 30)


def test_no_rows_no_work():
    assert loss(n=0, X=None, y=None, out=None) == 0
    assert gradient(n=0, X=None, y=None, out=None, gx=None, weight=None) == -1


def test_embed_refuses():
    def rows(table=AT, dtype=_lib.LBT_F32, n=10, f=8, tokens=Y, width=8, t=5, out=OUT):
        return L.lbt_embed_rows(None, table, dtype, n, f, tokens, width, t, 1.0, out)

    def grad(g=AT, dtype=_lib.LBT_F32, tokens=Y, width=8, t=5, f=8, n=10, add=0, out=OUT, ws=WS, size=BIG):
        return L.lbt_embed_rows_gradient(None, g, dtype, tokens, width, t, f, n, 1.0, add, out, ws, size)

    for call in (rows, grad):
        for arguments, message in ((dict(dtype=_lib.LBT_F64), b"dtype"), (dict(n=0), b"shape"), (dict(f=0), b"shape"),
                                   (dict(t=-1), b"shape"), (dict(t=1 << 31), b"shape"), (dict(n=1 << 30, f=1 << 20), b"shape"),
                                   (dict(width=2), b"tokens"), (dict(tokens=None), b"null"), (dict(out=None), b"null"),
                                   (dict(out=ODD), b"aligned")):
            assert call(**arguments) == -1, arguments
            assert message in L.lbt_last_error(), arguments
    assert rows(table=ODD) == -1 and rows(table=None) == -1
    assert grad(g=ODD) == -1 and grad(g=None) == -1
    assert rows(t=0, tokens=None, out=None) == 0
    assert grad(t=0, add=1, g=None, tokens=None) == 0
    need = L.lbt_embed_rows_gradient_workspace_bytes(5, 8, 10, _lib.LBT_F32)
    assert need > 0 and grad(size=need - 1) == -3 and grad(ws=None) == -3 and grad(ws=ODD) == -3
    assert L.lbt_embed_rows_gradient_workspace_bytes(5, 8, 10, _lib.LBT_F64) == 0
    assert L.lbt_embed_rows_gradient_workspace_bytes(0, 8, 10, _lib.LBT_F32) > 0


def inside(a, by=16):
    return C.c_void_p(a.value + by)


def test_overlaps_are_refused():
    """Ten rows of 8 values of 2 bytes: 160 bytes of X, 1600 of weight, 40 of the loss."""
    for call, arguments in ((loss, dict(out=inside(AT, 156))), (loss, dict(out=inside(Y, 64))), (loss, dict(ws=inside(W, 256), size=BIG)),
                            (loss, dict(bias=inside(OUT))), (gradient, dict(gx=AT)), (gradient, dict(gw=inside(W, 1584))),
                            (gradient, dict(gx=inside(GW))), (gradient, dict(out=inside(GX, 144))), (gradient, dict(w=inside(OUT, 36))),
                            (gradient, dict(bias=GB, gb=GB))):
        assert call(**arguments) == -1 and b"overlap" in L.lbt_last_error(), arguments
    # side by side is apart: the next check, that of the workspace, is reached
    assert gradient(gx=inside(AT, 160), gw=inside(W, 1600)) == -3
    rows, grad = L.lbt_embed_rows, L.lbt_embed_rows_gradient
    assert rows(None, AT, _lib.LBT_F32, 10, 8, Y, 8, 5, 1.0, inside(AT, 304)) == -1 and b"overlap" in L.lbt_last_error()
    assert grad(None, AT, _lib.LBT_F32, Y, 8, 5, 8, 10, 1.0, 1, AT, WS, BIG) == -1 and b"overlap" in L.lbt_last_error()
    assert grad(None, AT, _lib.LBT_F32, Y, 8, 5, 8, 10, 1.0, 1, OUT, inside(OUT), BIG) == -1 and b"overlap" in L.lbt_last_error()


def test_native_calls_leave_what_they_do_not_take():
    """No tensor, one on the host, a type or a shape of another kind: None, and the Python form says what is wrong."""
    import torch

    host = _lib._host
    table, tokens = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int64)
    for a, b in ((table, tokens), (table.numpy(), tokens), (table, [1, 2]), (None, None)):
        assert host.embed_rows(a, b, 0, 0, 0, 1.0) is None
        assert host.embed_rows_gradient(a, b, None, 0, 0, 0, 0, 4, 1.0) is None
        assert host.linear_log_loss(a, a, b, None, None, 0, 0, 0, 0) is None
        assert host.linear_log_loss_gradient(a, a, b, None, None, 0, 0, 0, 0, None) is None
    for scale in ("1", None, [1]):
        assert host.embed_rows(table, tokens, 0, 0, 0, scale) is None
    with pytest.raises(TypeError):
        host.embed_rows(table, tokens)
    for call in (host.embed_rows_gradient, host.linear_log_loss, host.linear_log_loss_gradient):
        with pytest.raises(TypeError):
            call(table, tokens)


def test_workspaces_of_many_rows():
    """Rows come in parts: millions of them take the scratch of one part, and no piece of the gradient passes 4 GiB."""
    q = L.lbt_linear_log_loss_workspace_bytes
    for dtype, size in ((_lib.LBT_BF16, 2), (_lib.LBT_F16, 2), (_lib.LBT_F32, 4)):
        for gradient in (0, 1, 2):
            for n, f, k in ((10000000, 100, 8), (2000000, 200, 8), (1 << 24, 28, 2), (1 << 30, 1, 1)):
                assert 0 < q(n, f, k, dtype, gradient) < (1 << 30), (n, f, k, dtype, gradient)
            # ten times the rows: the same but for what the parts' sizes differ by
            assert q(10000000, 100, 8, dtype, gradient) <= q(1000000, 100, 8, dtype, gradient) * 1.2
            # G and its exponentials, the tops and totals, X in planes twice and the sums of its gradient, and those of grad_weight
            weights = 4 * 131072 * 1024
            assert q(4000000, 1024, 131072, dtype, gradient) < (4 << 30) + (1 << 31) + 2 * (2 << 30) + (4 << 30) + (1 << 29) + weights


def test_the_largest_shapes():
    q, e = L.lbt_linear_log_loss_workspace_bytes, L.lbt_embed_rows_gradient_workspace_bytes
    for most, size in ((1 << 30, lambda v: q(v, 1, 1, _lib.LBT_BF16, 0)), ((1 << 30) - 64, lambda v: q(1, 1, v, _lib.LBT_BF16, 0)),
                       (1 << 20, lambda v: q(1, v, 1, _lib.LBT_BF16, 0)), (1 << 30, lambda v: e(v, 1, 1, _lib.LBT_BF16)),
                       ((1 << 30) - 64, lambda v: e(1, 1, v, _lib.LBT_BF16)), (1 << 24, lambda v: e(1, v, 1, _lib.LBT_BF16))):
        assert size(most) > 0 and size(most + 1) == 0
    assert loss(k=(1 << 30) - 63) == -1 and b"shape" in L.lbt_last_error()
    assert L.lbt_embed_rows(None, AT, _lib.LBT_BF16, (1 << 30) - 63, 1, Y, 8, 5, 1.0, OUT) == -1 and b"shape" in L.lbt_last_error()


def test_nothing_overlaps_an_empty_array():
    """No rows, no tokens: their addresses are not looked at, wherever they point. The next check, that of the workspace, is reached."""
    assert gradient(n=0, X=inside(GW), gx=inside(W), y=inside(GW, 32), out=inside(W, 48), w=inside(GW, 64)) == -3
    assert b"workspace" in L.lbt_last_error()
    grad = L.lbt_embed_rows_gradient
    assert grad(None, inside(OUT), _lib.LBT_F32, inside(OUT, 64), 8, 0, 8, 10, 1.0, 0, OUT, None, 0) == -3
    assert b"workspace" in L.lbt_last_error()


def test_the_least_workspace():
    q, least = L.lbt_linear_log_loss_workspace_bytes, 4
    for dtype in (_lib.LBT_BF16, _lib.LBT_F16, _lib.LBT_F32):
        for kind in (0, 1, 2):
            for n, f, k in ((10, 8, 100), (8192, 4096, 131072), (4096, 1000, 30000), (1, 1024, 32768), (300000, 64, 5000)):
                assert 0 < q(n, f, k, dtype, least + kind) <= q(n, f, k, dtype, kind), (dtype, kind, n, f, k)
        # X, its planes and sums, tops and totals, and those 128 MiB of G and 64 of weights
        assert q(8192, 4096, 131072, dtype, least + 1) < (7 << 27) and q(8192, 4096, 131072, dtype, 1) > (5 << 28)
        assert q(10, 8, 100, dtype, 7) == 0 and q(10, 0, 100, dtype, least) == 0
    need, small = q(8192, 4096, 131072, _lib.LBT_BF16, 1), q(8192, 4096, 131072, _lib.LBT_BF16, least + 1)
    assert gradient(n=8192, f=4096, k=131072, ws=WS, size=small - 1) == -3 and str(need).encode() in L.lbt_last_error()
