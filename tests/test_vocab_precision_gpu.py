"""How exact the gradients of bf16 inputs are, value by value against 64 bits.

Errors of a gradient's value, with S the sum of the sizes of its terms w (p + q) |operand|:
  p               logits to 1e-5 (fp32 sums, operands as they are), so p to 1e-5 of itself; the sum
                  over the terms in fp32: together at most 2e-5 S, what the losses are held to
  G = w (p - q)   in one fp16 part (bf16 gradients): 2^-11 of itself; in two parts (fp32 gradients): 2^-23, within
                  the 2e-5
  bf16 result     one rounding, 2^-8 of the value
An fp16 part's values lie 2^-24 apart at least, so it is off by 2^-25 beside a largest value of 2^13 (w H; W of
2^14, G of 2^14): 2^-38 of the largest, in two parts 2^-49.  FLOOR adds that up over the terms.
"""
import numpy as np
import pytest

from _gpu import DB
from dreamcompiler_amd import hip
from test_vocab_gpu import DT, F32_TOL, Loss, close, fetch, ints, store

FLOOR = {"bf16": 2.0 ** -38, "f32": 2.0 ** -49}


def gradients(c, grad, accumulate=False, extra=0):
    """dH and dW of a Loss, and its loss and lse, as 64-bit values; `extra` bytes above the least workspace."""
    size = max(c.least(0), c.least(1)) + extra
    ws = DB(size)
    loss, lse = DB.empty((c.N,), np.float32), DB.empty((c.N,), np.float32)
    r = np.random.default_rng(9)
    shapes = ((c.N, c.D), (c.V, c.D))
    old = [r.standard_normal(s) * c.dloss.max() if accumulate else np.full(s, np.nan) for s in shapes]
    bufs = [store(x, grad, c.ld) for x in old]
    c.fwd(loss, lse, ws, size)
    c.bwd(lse, c.dlb, bufs[0][0], c.ld, accumulate, bufs[1][0], c.ld, accumulate, DT[grad], ws, size)
    got = [fetch(b, s, grad, c.ld)[0] for (b, _), s in zip(bufs, shapes)]
    return (*got, loss.numpy().astype(np.float64), lse.numpy().astype(np.float64),
            [x if accumulate else 0.0 for _, x in bufs])


def sizes(c, lse, grad):
    """S of every value of dH and dW, and what lies below their parts."""
    k = c.keep
    inv = c.scale if c.K is None else 1 / c.T
    w = np.abs(c.dloss[:, None]) * (c.scale if c.K is None else c.T) * k[:, None]
    P = w[k] * (np.exp(inv * (c.H[k] @ c.W.T) - lse[k, None]) + c.q[k])
    dH = np.zeros((c.N, c.D))
    dH[k] = P @ np.abs(c.W)
    H = np.where(k[:, None], np.abs(c.H), 0.0)
    low = w * (np.abs(c.W).sum(0) + 2 * np.abs(c.W).max()), (w * H).sum(0) + k.sum() * (w * H).max(initial=0.0)
    return (dH, P.T @ H[k]), [FLOOR[grad] * x + 2.0 ** -126 for x in low]


def check(c, grad, accumulate=False, extra=0, part=2.0 ** -11):
    """All four results to the bounds above; `part` is what one part of G loses."""
    dH, dW, loss, lse, old = gradients(c, grad, accumulate, extra)
    ref = c.ref()
    close(loss, ref[0], F32_TOL, floor=1.0)
    close(lse, ref[1], F32_TOL, floor=1.0)
    for name, got, want, S, low, add in zip(("dH", "dW"), (dH, dW), ref[2:], *sizes(c, ref[1], grad), old):
        want = want + add
        bound = F32_TOL * S + 2.0 ** -23 * np.abs(want) + low
        if grad == "bf16":
            bound = 2.0 ** -8 * np.abs(want) + (1 + 2.0 ** -8) * (bound + part * S)
        off = np.abs(got - want)
        worst = np.unravel_index(np.argmax(off / bound), off.shape)
        assert np.isfinite(got).all() and (off <= bound).all(), (name, worst, off[worst], bound[worst])


@pytest.mark.gpu
@pytest.mark.parametrize("grad", ["f32", "bf16"])
@pytest.mark.parametrize("K,T", [(None, 1.0), (6, 2.0)])
@pytest.mark.parametrize("N,V,D", [(5, 700, 40), (17, 300, 64), (70, 1000, 72), (200, 2000, 130), (520, 4100, 72),
                                   (700, 700, 1100)])
def test_gradients_value_by_value(N, V, D, K, T, grad):
    check(Loss(N, V, D, "bf16", K=K, T=T, pad=0.2), grad)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [4, 5, 16, 17])
def test_gradients_do_not_get_coarser_with_a_row_more(N):
    """Over a table of more than 2^22 values."""
    check(Loss(N, 70000, 64, "bf16"), "f32")
    check(Loss(N, 70000, 64, "bf16"), "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("N", [1, 4, 5, 16])
@pytest.mark.parametrize("V,D", [(300, 64), (70000, 64)])
def test_few_rows_keep_G_in_floats(N, V, D):
    check(Loss(N, V, D, "bf16", seed=1), "bf16", part=0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("grad", ["f32", "bf16"])
def test_gradients_of_many_rows_with_one_target(grad):
    """Rows whose weights are about 0.502 of the largest (in bf16 the worst of all to round, always upwards), their
    target the same and hopeless, H and W of one sign: what is lost of G would add up."""
    N, V, D = 200, 300, 64
    c = Loss(N, V, D, "bf16", seed=3)
    r = np.random.default_rng(8)
    W = r.random((V, D)) * 0.02
    W[7] = -0.3
    c.Hb, c.H = store(np.abs(r.standard_normal((N, D))) + 0.1, "bf16")
    c.Wb, c.W = store(W, "bf16")
    c.dloss = (0.501953125 + 2.0 ** -14 * (1 + r.random(N))).astype(np.float32)
    c.dloss[0] = 1.0
    c.dlb = DB.from_numpy(c.dloss)
    c.ids = ints(np.full(N, 7))
    c.q[:] = 0
    c.q[:, 7] = 1
    check(c, grad)


@pytest.mark.gpu
@pytest.mark.parametrize("weights", ["zero", "wide", "huge", "one row"])
@pytest.mark.parametrize("grad", ["f32", "bf16"])
def test_gradients_keep_rows_of_any_weight(weights, grad):
    """dH of a row to its own size, however small its weight beside the others'."""
    N, V, D = 150, 400, 48
    c = Loss(N, V, D, "bf16", seed=6, pad=0.1)
    r = np.random.default_rng(7)
    c.dloss = {"zero": np.zeros(N), "wide": np.ldexp(r.standard_normal(N), r.integers(-90, 1, N)),
               "huge": np.ldexp(1 + r.random(N), 100), "one row": np.eye(N)[11]}[weights].astype(np.float32)
    c.dlb = DB.from_numpy(c.dloss)
    dH, dW, _, lse, _ = gradients(c, grad)
    ref = c.ref()
    S, _ = sizes(c, ref[1], grad)
    tol = F32_TOL + (2.0 ** -8 + 2.0 ** -11 if grad == "bf16" else 0)
    rows = np.maximum(S[0].max(1, keepdims=True), 2.0 ** -110)
    assert (np.abs(dH - ref[2]) <= 2 * tol * rows).all()
    close(dW, ref[3], 2 * tol, floor=max(S[1].max(), 2.0 ** -110))


@pytest.mark.gpu
@pytest.mark.parametrize("k", [-60, 0, 60])
@pytest.mark.parametrize("weights", ["any", "zero"])
def test_gradients_of_operands_of_any_scale(k, weights):
    """H 2^k and W 2^-k: bf16 has fp32's range."""
    c = Loss(70, 300, 40, "bf16", seed=3)
    if weights == "zero":
        c.dloss[:] = 0
        c.dlb = DB.from_numpy(c.dloss)
    c.Hb, c.H = store(np.ldexp(c.H, k), "bf16")
    c.Wb, c.W = store(np.ldexp(c.W, -k), "bf16")
    for grad in ("f32", "bf16"):
        check(c, grad)


@pytest.mark.gpu
@pytest.mark.parametrize("N,V,D", [(70, 1000, 100), (40, 300, 1030)])
def test_products_whose_low_parts_all_add_up(N, V, D):
    """Every operand 2^e (1 + 2^-11): its high part is 2^e, and the product of the low parts, 2^-22 of each term and
    the one that is left out, has one sign in all of them.  2^-22 of a logit of 20 is 5e-6, within what fp32 results
    are held to."""
    c = Loss(N, V, D, "f32", seed=2)
    r = np.random.default_rng(1)
    one = 1 + 2.0 ** -11
    c.Hb, c.H = store(np.ldexp(one, r.integers(-3, 1, (N, D))), "f32")
    c.Wb, c.W = store(np.ldexp(one, r.integers(-3, 1, (V, 1)) * np.ones((1, D), int) - int(np.log2(D)) + 4), "f32")
    assert 5 < (c.H @ c.W.T).max() < 25
    check(c, "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,grad", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("k,weight", [(120, -110), (-60, 60)])
def test_large_operands_of_small_weights(k, weight, dtype, grad):
    """w H is within fp32 where H's sum over the rows is not."""
    c = Loss(400, 60, 40, dtype, seed=3)
    c.Hb, c.H = store(np.ldexp(np.abs(c.H), k), dtype)
    c.Wb, c.W = store(np.ldexp(c.W, -k), dtype)
    c.ids = ints(np.full(c.N, 3))
    c.q[:] = 0
    c.q[:, 3] = 1
    c.dloss = np.ldexp(c.dloss, weight).astype(np.float32)
    c.dlb = DB.from_numpy(c.dloss)
    dH, dW, *_ = gradients(c, grad)
    ref = c.ref()
    S, low = sizes(c, ref[1], grad)
    tol = F32_TOL + (2.0 ** -8 + 2.0 ** -11 if grad == "bf16" else 0)
    assert np.isfinite(dW).all() and (np.abs(dW - ref[3]) <= 2 * tol * S[1] + low[1]).all()
    assert np.isfinite(dH).all() and (np.abs(dH - ref[2]) <= 2 * tol * S[0] + low[0]).all()
