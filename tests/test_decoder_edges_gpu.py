"""The operators around a decoder's attention where their sizes, addresses and values are at an edge.  Tolerances are
those of the operators' own tests."""
import numpy as np
import pytest

from _decoder import TYPE, U, UB, attention, within
from dreamcompiler_amd import hip
from test_paged_attention_gpu import KINDS, Case

SAME = [("f32", "f32"), ("bf16", "bf16")]


# ------------------------------------------------------------------------------ attention

def near(x, b, heads=slice(None)):
    """Sequence b's results for these heads, by the bounds of the attention's own tests."""
    o, lse, A = (y[heads] for y in attention(x.Q.value[b], x.value[0][b], x.value[1][b], x.scale))
    dz = (2 * x.D ** 0.5 + 8) * U * A
    bf16 = x.dtype == "bf16"
    tol = ((2 * dz + 64 * U + (2.0 ** -16 if bf16 else 0)) * np.abs(x.value[1][b]).max())[:, None]
    within(x.O.get()[b][heads], o, tol + (UB * (np.abs(o) + tol) if bf16 else 0))
    within(x.lse.numpy()[b][heads], lse, dz + 64 * U + 2 * U * np.abs(lse))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", SAME)
@pytest.mark.parametrize("Hq,Hk,D", [(4, 2, 64), (20, 1, 128), (3, 1, 48)])
def test_no_score_but_values_that_are_not_finite(Hq, Hk, D, dtype, kind):
    """Sequences whose scores are all -infinity are empty rows, whatever their values hold: of one chunk, of a few
    that one wave joins, and of many."""
    def away(q, K, V):
        q[:] = np.abs(q) + 0.1
        for b, (k, v) in enumerate(zip(K, V)):
            if b % 2 == 0:
                k[:] = -np.inf
                v[::3], v[1::3] = np.inf, np.nan

    for T in (40, 2000, 20000):
        x = Case(dtype, kind, [T, 33, T // 2, 1], Hq, Hk, D, 16, change=away).run()
        got, L = x.O.get(), x.lse.numpy()
        for b in (0, 2):
            assert (got[b] == 0).all() and (L[b] == -np.inf).all()
        for b in (1, 3):
            near(x, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
def test_queries_at_infinity(dtype, kind):
    """Keys above zero and a query of -infinity: no score; where one value of it is +infinity beside: NaN.  The other heads
    and sequences stay as they are."""
    def far(q, K, V):
        for k in K:
            k[:] = np.abs(k) + 0.5
        q[0, 1, 5] = -np.inf
        q[2, :] = -np.inf
        q[0, 2, 3], q[0, 2, 9] = -np.inf, np.inf

    x = Case(dtype, kind, [70, 40, 1500], 4, 2, 64, 16, change=far).run()
    got, L = x.O.get(), x.lse.numpy()
    for b, h in ((0, 1), (2, slice(None))):
        assert (got[b, h] == 0).all() and (L[b, h] == -np.inf).all()
    assert np.isnan(got[0, 2]).all() and np.isnan(L[0, 2])
    for b, heads in ((0, [0, 3]), (1, [0, 1, 2, 3])):
        near(x, b, heads)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
def test_one_chunk_needs_no_workspace(dtype, kind):
    """A window that is not split, over sequences that would be."""
    x = Case(dtype, kind, [3000, 5, 2999], 4, 2, 64, 16, window=300)
    assert hip.paged_attention_plan(TYPE[kind], 3, 4, 2, 64, x.max_len, 300)[1] == 1 and x.size > 0
    x.run().check()
    want = x.values()
    x.wipe()
    x.ws, x.size = None, 0
    x.run().check()
    assert all(np.array_equal(a, b) for a, b in zip(x.values(), want))
