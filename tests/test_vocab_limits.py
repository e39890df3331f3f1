"""The largest sizes: what the embedding's gradient and the vocabulary losses refuse because a launch could not hold it
(before anything is written), and large ones that they take."""
import numpy as np
import pytest

from _gpu import DB
from dreamcompiler_amd import hip
from test_vocab_gpu import ints
from test_vocab_refusals import LOSSES, emb_bwd, raises


@pytest.mark.parametrize("N", [2 ** 28 - 15, 2 ** 28, 2 ** 30])
def test_embedding_gradient_of_more_tokens_than_a_launch_holds(N):
    with raises("shape"):
        emb_bwd(N=N)


def test_embedding_gradient_of_as_many_as_it_holds():
    with raises("workspace of"):
        emb_bwd(N=2 ** 28 - 16, size=0)


@pytest.mark.parametrize("f", LOSSES)
def test_losses_of_more_rows_than_a_launch_holds(f):
    for shape in (dict(N=2 ** 25 + 1), dict(N=2 ** 30), dict(N=2 ** 21, D=2 ** 15, V=70)):
        with raises("shape"):
            f(**shape)
    for shape in (dict(N=2 ** 25), dict(N=2 ** 20, D=2 ** 15, ldh=2 ** 15, ldw=2 ** 15, lddh=2 ** 15, lddw=2 ** 15)):
        if f.__name__.endswith("fwd"):
            shape = {k: v for k, v in shape.items() if k not in ("lddh", "lddw")}
        with raises("workspace of"):
            f(size=0, **shape)


@pytest.mark.gpu
@pytest.mark.parametrize("accumulate", [False, True])
def test_embedding_gradient_of_2_25_tokens(accumulate):
    """Sums of up to 130000 values of size up to 8 are exact in fp32."""
    N, V, D = (1 << 25) + 5, 300, 2
    r = np.random.default_rng(0)
    ids = r.integers(-1, V, N, dtype=np.int32)
    dY = r.integers(-8, 9, (N, D)).astype(np.float32)
    size = hip.embedding_bwd_workspace(N, V, D)
    ws, ib, yb = DB(size), ints(ids), DB.from_numpy(dY)
    dW = DB.from_numpy(np.full((V, D), 3, np.float32))
    hip.embedding_bwd(hip.F32, N, V, D, 1.0, ib, yb, D, dW, D, hip.F32, accumulate, ws, size)
    want = np.stack([np.bincount(ids + 1, dY[:, d], V + 1)[1:] for d in range(D)], 1) + (3 if accumulate else 0)
    assert (dW.numpy() == want).all()
    for b in (ws, ib, yb, dW):
        b.free()


@pytest.mark.gpu
def test_teacher_of_more_rows_than_one_dimension_holds():
    """2^22 rows and some: the launches of one work-group a row have a second dimension.  Rows repeat with a period."""
    N, V, D, K, P = (1 << 22) + 1000, 9, 4, 2, 1024
    r = np.random.default_rng(0)
    rep = lambda x: np.ascontiguousarray(np.resize(x, (N,) + x.shape[1:]))  # noqa: E731
    H, W = r.standard_normal((P, D)).astype(np.float32), r.standard_normal((V, D)).astype(np.float32)
    ids = r.integers(-1, V, (P, K)).astype(np.int32)
    logit = r.standard_normal((P, K)).astype(np.float32)

    def run(H, ids, logit):
        n = len(H)
        Hb, Wb, ib, lb = DB.from_numpy(H), DB.from_numpy(W), ints(ids), DB.from_numpy(logit)
        size = max(hip.linear_distill_workspace(hip.F32, n, V, D, K, b) for b in (0, 1))
        ws = DB(size)
        loss, lse = DB.empty((n,), np.float32), DB.empty((n,), np.float32)
        dH, dW = DB.empty((n, D), np.float32), DB.empty((V, D), np.float32)
        a = (hip.F32, n, V, D, K, 1.0, Hb, D, Wb, D, ib, lb)
        hip.linear_distill_fwd(*a, loss, lse, ws, size)
        hip.linear_distill_bwd(*a, lse, None, dH, D, False, dW, D, False, hip.F32, ws, size)
        out = [x.numpy().astype(np.float64) for x in (loss, lse, dH, dW)]
        for b in (Hb, Wb, ib, lb, ws, loss, lse, dH, dW):
            b.free()
        return out

    few, many = run(H, ids, logit), run(rep(H), rep(ids), rep(logit))
    for a, b in zip(few[:3], many[:3]):   # the products' tiles may differ
        assert np.abs(rep(a) - b).max() <= 4e-5 * max(1.0, np.abs(a).max())
    # dW: 4096 times and the first 1000 rows once more, in fp32 sums; those rows' part is below a period's own
    G = few[3] * (N // P)
    part = run(H[:N % P], ids[:N % P], logit[:N % P])[3] if N % P else 0.0
    assert np.abs(G + part - many[3]).max() <= 2e-5 * N * np.abs(H).max()
