"""What the embedding and the vocabulary losses refuse, before they touch a device: no GPU needed.
The addresses are never read."""
import pytest

from dreamcompiler_amd import hip

P, ODD = 1 << 20, (1 << 20) + 8
NAN, INF = float("nan"), float("inf")
BIG = 1 << 40


def raises(match):
    return pytest.raises(hip.DreamHipError, match=match)


def emb_fwd(dt=0, N=4, V=9, D=8, scale=1.0, ids=P, W=P, ldw=8, Y=P, ldy=8):
    hip.embedding_fwd(dt, N, V, D, scale, ids, W, ldw, Y, ldy)


def emb_bwd(dt=0, N=4, V=9, D=8, scale=1.0, ids=P, dY=P, lddy=8, dW=P, lddw=8, gt=0, ws=P, size=BIG):
    hip.embedding_bwd(dt, N, V, D, scale, ids, dY, lddy, dW, lddw, gt, False, ws, size)


def xent_fwd(dt=0, N=4, V=9, D=8, scale=1.0, H=P, ldh=8, W=P, ldw=8, t=P, loss=P, ws=P, size=BIG):
    hip.linear_xent_fwd(dt, N, V, D, scale, H, ldh, W, ldw, t, loss, None, ws, size)


def xent_bwd(dt=0, N=4, V=9, D=8, scale=1.0, H=P, ldh=8, W=P, ldw=8, t=P, lse=P, dH=P, lddh=8, dW=P, lddw=8, gt=0,
             ws=P, size=BIG):
    hip.linear_xent_bwd(dt, N, V, D, scale, H, ldh, W, ldw, t, lse, None, dH, lddh, False, dW, lddw, False, gt, ws,
                        size)


def distill_fwd(dt=0, N=4, V=9, D=8, K=2, scale=1.0, H=P, ldh=8, W=P, ldw=8, t=P, z=P, loss=P, ws=P, size=BIG):
    hip.linear_distill_fwd(dt, N, V, D, K, scale, H, ldh, W, ldw, t, z, loss, None, ws, size)


def distill_bwd(dt=0, N=4, V=9, D=8, K=2, scale=1.0, H=P, ldh=8, W=P, ldw=8, t=P, z=P, lse=P, dH=P, lddh=8, dW=P,
                lddw=8, gt=0, ws=P, size=BIG):
    hip.linear_distill_bwd(dt, N, V, D, K, scale, H, ldh, W, ldw, t, z, lse, None, dH, lddh, False, dW, lddw, False,
                           gt, ws, size)


LOSSES = [xent_fwd, xent_bwd, distill_fwd, distill_bwd]
ALL = [emb_fwd, emb_bwd] + LOSSES


@pytest.mark.parametrize("f", ALL)
def test_types_and_shapes(f):
    for dt in (-1, 2, 7):
        with raises("dtype"):
            f(dt=dt)
    most = 1 << 20 if f in LOSSES else 1 << 24
    for bad in (dict(N=-1), dict(V=0), dict(V=-3), dict(D=0), dict(D=most + 1), dict(N=2 ** 31 - 1),
                dict(V=2 ** 31 - 1)):
        with raises("shape"):
            f(**bad)


@pytest.mark.parametrize("f,names", [(emb_fwd, "ldw ldy"), (emb_bwd, "lddy lddw"), (xent_fwd, "ldh ldw"),
                                     (xent_bwd, "ldh ldw lddh lddw"), (distill_fwd, "ldh ldw"),
                                     (distill_bwd, "ldh ldw lddh lddw")])
def test_leading_dimensions(f, names):
    for n in names.split():
        for ld in (7, 0, -8):
            with raises("leading dimension"):
                f(**{n: ld})


@pytest.mark.parametrize("f,names", [(emb_fwd, "ids W Y"), (emb_bwd, "ids dY dW"), (xent_fwd, "H W loss ws t"),
                                     (xent_bwd, "H W lse ws t"), (distill_fwd, "H W t z loss ws"),
                                     (distill_bwd, "H W t z lse ws")])
def test_null_pointers(f, names):
    for n in names.split():
        with raises("null"):
            f(**{n: None})
    if f is emb_bwd:
        with raises("null"):
            f(N=3000, ws=None)


@pytest.mark.parametrize("f", LOSSES)
def test_scale_and_temperature(f):
    for s in (0.0, -1.0, NAN, INF):
        with raises("finite"):
            f(scale=s)
    if f in (distill_fwd, distill_bwd):
        for s in (1e-39, 1e30):     # 1 / T or T^2 past fp32's range
            with raises("finite"):
                f(scale=s)


@pytest.mark.parametrize("f", [emb_fwd, emb_bwd])
def test_embedding_scale(f):
    for s in (NAN, INF, -INF):
        with raises("finite"):
            f(scale=s)


@pytest.mark.parametrize("f", [emb_bwd, xent_bwd, distill_bwd])
def test_gradient_type(f):
    for dt, gt in ((0, 1), (0, 5), (1, -1)):
        with raises("grad_type"):
            f(dt=dt, gt=gt)


@pytest.mark.parametrize("f,need", [
    (emb_bwd, lambda n: hip.embedding_bwd_workspace(n, 9, 8)),
    (xent_fwd, lambda n: hip.linear_xent_workspace(0, n, 9, 8, 0)),
    (xent_bwd, lambda n: hip.linear_xent_workspace(0, n, 9, 8, 1)),
    (distill_fwd, lambda n: hip.linear_distill_workspace(0, n, 9, 8, 2, 0)),
    (distill_bwd, lambda n: hip.linear_distill_workspace(0, n, 9, 8, 2, 1))])
def test_workspaces(f, need):
    for n in (1, 16, 17, 32, 33, 3000):
        if need(n) > 0:
            with raises("workspace of"):
                f(N=n, size=need(n) - 1)
            with raises("workspace not 16-byte aligned"):
                f(N=n, ws=ODD)


def test_entries_of_a_teacher():
    for f in (distill_fwd, distill_bwd):
        with raises("K=-1"):
            f(K=-1)


def test_workspace_queries_of_nothing_and_of_much():
    """A shape that the call refuses needs nothing; the least workspace grows with its operands."""
    assert hip.linear_xent_workspace(0, 100, 50000, 512, 1) > 2 * 100 * 512 * 2
    for dt in (0, 1):
        for b in (0, 1):
            a = [hip.linear_xent_workspace(dt, n, 50000, 512, b) for n in (16, 100, 1000, 10000)]
            assert a[1:] == sorted(a[1:]) and all(x > 0 for x in a)
