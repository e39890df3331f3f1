"""Distillation from teachers of many entries a row, with tokens that occur more than once."""
import numpy as np
import pytest

from _gpu import DB
from dreamcompiler_amd import hip
from test_vocab_gpu import DT, Loss, ints, run_loss, store
from test_vocab_gpu import test_graphs_on_other_streams as graphs_on_other_streams
from test_vocab_precision_gpu import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,grad", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("N,V,K", [(40, 50, 200), (3, 50, 200), (40, 4097, 1100), (9, 4097, 1100), (20, 300, 128), (20, 300, 129),
                                   (17, 13000, 3000), (16, 13000, 300), (40, 8192, 8192),
                                   (11000, 50, 130)])
def test_many_entries(N, V, K, dtype, grad):
    check(Loss(N, V, 40, dtype, K=K, T=2.0, pad=0.2, seed=K), grad)


@pytest.mark.parametrize("N", [6, 60])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_one_token_in_all_entries(N, dtype):
    """Its probabilities add up to one, whatever their order; twice the same bits."""
    c = Loss(N, 70, 24, dtype, K=600, seed=1)
    c.idx[:] = 69
    c.ids = ints(c.idx)
    top = np.random.default_rng(0).standard_normal((N, 600)).astype(np.float32)
    c.top = DB.from_numpy(top)
    e = np.exp(top.astype(np.float64) - top.max(1, keepdims=True))
    c.ok, c.keep, c.qk = np.ones_like(c.ok), np.ones(N, bool), e / e.sum(1, keepdims=True)
    c.q = np.zeros_like(c.q)
    c.q[:, 69] = 1
    check(c, dtype)
    for a, b in zip(run_loss(c), run_loss(c)):
        assert (a == b).all()


@pytest.mark.parametrize("N", [6, 60])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_logit_that_is_no_number(N, bad):
    """Its row's loss and gradient are NaN, no other row's."""
    V, D, K = 300, 24, 200
    c = Loss(N, V, D, "f32", K=K, seed=1)
    clean = run_loss(c)
    top = c.top.numpy((N, K), np.float32)
    n = int(np.nonzero(c.keep)[0][2])
    k = int(np.nonzero(c.ok[n])[0][1])
    top[n, k] = bad
    c.top = DB.from_numpy(top)
    size = max(c.least(0), c.least(1))
    ws = DB(size)
    loss, lse = DB.empty((N,), np.float32), DB.empty((N,), np.float32)
    dH = store(np.zeros((N, D)), "f32")[0]
    c.fwd(loss, lse, ws, size)
    c.bwd(lse, c.dlb, dH, D, False, None, D, False, DT["f32"], ws, size)
    l, g = loss.numpy(), dH.numpy((N, D), np.float32)
    others = np.arange(N) != n
    assert np.isnan(l[n]) and np.isnan(g[n]).all()
    assert (l[others] == clean[0][others]).all() and (g[others] == clean[2][others]).all()


@pytest.mark.parametrize("N", [8, 512])
def test_time_does_not_grow_with_the_square_of_the_entries(N):
    """8 times the entries take at most 24 times as long; looking through the row for each, 43 and 31 times: 19.8 ms
    for 8192 entries of 512 rows and 638 us for 1024."""
    V, D = 32000, 64
    r = np.random.default_rng(0)
    H, W = store(r.standard_normal((N, D)), "bf16")[0], store(r.standard_normal((V, D)), "bf16")[0]
    times = []
    for K in (1024, 8192):
        ids = ints(np.argsort(r.random((N, V)), 1)[:, :K])
        top = DB.from_numpy(r.standard_normal((N, K)).astype(np.float32))
        size = max(hip.linear_distill_workspace(hip.BF16, N, V, D, K, b) for b in (0, 1))
        ws = DB(size)
        loss, lse = DB.empty((N,), np.float32), DB.empty((N,), np.float32)
        dH, dW = DB.empty((N, D), np.uint16), DB.empty((V, D), np.uint16)
        a = (hip.BF16, N, V, D, K, 1.0, H, D, W, D, ids, top)

        def step():
            hip.linear_distill_fwd(*a, loss, lse, ws, size)
            hip.linear_distill_bwd(*a, lse, None, dH, D, False, dW, D, False, hip.BF16, ws, size)

        step()
        hip.sync()
        best = np.inf
        for _ in range(3):
            with hip.Timer() as timer:
                for _ in range(4):
                    step()
            best = min(best, timer.ms)
        times.append(best)
    assert times[1] <= 24 * times[0], times


@pytest.mark.parametrize("a,b", [((11000, 40, 24, "bf16", None), (300, 700, 130, "f32", 300)),
                                 ((11000, 40, 24, "f32", 20), (9, 700, 130, "bf16", 300)),
                                 ((1030, 8200, 72, "bf16", 200), (520, 4100, 72, "f32", None))])
def test_graphs(a, b):
    """The launches that only many rows or entries take, and wide tiles, recorded and replayed."""
    graphs_on_other_streams(a, b)
