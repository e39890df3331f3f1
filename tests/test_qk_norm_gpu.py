"""RMS norm of queries and keys with the rotation by position, and its gradient, against plain formulas
in 64 bits.

Tolerances (u = 2^-24, ub = 2^-8: the largest relative error of one rounding to fp32, to bf16).
 forward   the sum of D <= 1024 squares: up to 16 in a lane and six steps over lanes, 23 u, half of it after the
           root; root, quotient, two products: 4 u; a turned value is a sum of two such products with
           the table's (given) cosine and sine: 3 u of |y| + |y'| <= 2 max |y|.  Under 2 (12 + 4 + 3) u: 48 u
           of the row's largest y.  Then one rounding to the output's type.
 dx        x r to 16 u, dy g to 5 u, their mean over D: 25 u of the terms' mean size: under 64 u of
           r (max |dy g| + max |x r| mean |dy g x r|); one rounding to its type.
 dg        each term to 24 u of the products it is made of; a
           chain of additions is at most the rows of a lane (of 4096 waves), the 64 rows that
           meet in a work-group, 16 of 1024 work-groups, and 64: under (64 + min(rows, 520)) u of the terms' sizes.
"""
import numpy as np
import pytest

from _decoder import TYPE, U, UB, Strided, floats, ints, norm_rope, rope_table, within
from _gpu import DB
from dreamcompiler_amd import hip

EPS = 1e-6


def run(B, S, Hq, Hk, D, R, pairs, dtype, dout="f32", grad=None, pad=0, order=(0, 1, 2), out_order=(0, 2, 1),
        pos="rising", weights=True, accumulate=False, seed=0, eps=EPS, scale=1.0, same=False):
    r = np.random.default_rng(seed)
    grad = grad or dtype
    P = max(S + 5, 8)
    table = rope_table(P, R)
    where = {"rising": np.tile(np.arange(S), (B, 1)), "none": np.tile(np.arange(S), (B, 1)),
             "any": r.integers(-3, P + 3, (B, S)), "padding": np.full((B, S), -1)}[pos]
    if pos == "any" and where.size > 2:
        where.flat[0], where.flat[1] = 2 ** 31 - 1, -2 ** 31
    X = [Strided(scale * r.standard_normal((B, S, H, D)), dtype, order, pad) for H in (Hq, Hk)]
    dY = [Strided(r.standard_normal((B, S, H, D)), dout, out_order, pad) for H in (Hq, Hk)]
    g = [1 + 0.3 * r.standard_normal(D).astype(np.float32) for _ in range(2)]
    gb = [floats(x) if weights else None for x in g]
    gv = [x.astype(np.float64) if weights else 1.0 for x in g]
    out = [Strided(np.full((B, S, H, D), 7.0), dtype, out_order, pad) for H in (Hq, Hk)]
    dX = [Strided(np.full((B, S, H, D), 7.0), grad, order, pad) for H in (Hq, Hk)]
    old = r.standard_normal((2, D)).astype(np.float32)
    dg = [floats(x) for x in old]
    a = (TYPE[dtype], B, S, Hq, Hk, D, R, pairs, eps, None if pos == "none" else ints(where),
         floats(table) if R else None, P, X[0], X[0].strides, X[1], X[1].strides, *gb)
    hip.qk_norm_rope_fwd(*a, out[0], out[0].strides, out[1], out[1].strides)
    size = hip.qk_norm_rope_bwd_workspace(D)
    ws = DB(size)
    hip.qk_norm_rope_bwd(*a, TYPE[dout], dY[0], dY[0].strides, dY[1], dY[1].strides, TYPE[grad],
                         dX[0], dX[0].strides, dX[1], dX[1].strides, dg[0], dg[1], accumulate, ws, size)
    raws = []
    for i in range(2):
        if X[i].value.size == 0:
            continue
        ref = norm_rope(X[i].value, gv[i], where, table, R, pairs, eps)
        ok = ((where >= 0) & (where < P))[:, :, None, None]
        unturned = np.where(ok, norm_rope(X[i].value, gv[i], where * 0, table[:1] * 0 + 1, 0, pairs, eps), 0)
        tol = 48 * U * np.abs(unturned).max(-1, keepdims=True)
        within(out[i].get(), ref, tol + (UB * np.abs(ref) * (1 + UB) if dtype == "bf16" else 0))
        dx, dw, by, terms = norm_rope(X[i].value, gv[i], where, table, R, pairs, eps, dY[i].value)
        within(dX[i].get(), dx, 64 * U * by + (UB * (np.abs(dx) + 64 * U * by) if grad == "bf16" else 0))
        rows = B * S * (Hq, Hk)[i]
        tol = (64 + min(rows, 520)) * U * (terms + (np.abs(old[i]) if accumulate else 0))
        within(dg[i].numpy(), dw + (old[i] if accumulate else 0), tol)
        raws += [out[i].raw(), dX[i].raw(), dg[i].numpy()]
    return raws


SHAPES = [(1, 1, 1, 1, 1, 0), (1, 1, 32, 8, 128, 128), (2, 3, 5, 2, 7, 6), (1, 17, 12, 3, 80, 40), (3, 33, 4, 1, 96, 96),
          (2, 9, 3, 3, 100, 50), (1, 5, 2, 1, 256, 256), (1, 3, 2, 2, 300, 64), (1, 2, 1, 1, 1024, 1024),
          (2, 65, 8, 8, 64, 64), (1, 130, 6, 2, 32, 16), (4, 31, 16, 16, 128, 128), (2, 20, 4, 2, 192, 192),
          (1, 40, 8, 8, 128, 64), (1, 9, 16, 1, 16, 8), (1, 7, 3, 1, 72, 24), (2, 5, 10, 2, 512, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("dtype,dout,grad", [("f32", "f32", "f32"), ("bf16", "f32", "bf16"), ("bf16", "bf16", "bf16"),
                                             ("bf16", "bf16", "f32"), ("bf16", "f32", "f32")])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_norm_and_rotation(shape, dtype, dout, grad, pairs):
    run(*shape, pairs, dtype, dout, grad)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad,order,out_order", [(0, (1, 2, 0), (2, 0, 1)), (3, (0, 1, 2), (0, 2, 1)), (8, (2, 1, 0), (0, 1, 2)),
                                                 (1, (0, 2, 1), (1, 0, 2)), (16, (1, 0, 2), (2, 1, 0))])
def test_strides(pad, order, out_order, dtype):
    for D, R in ((64, 64), (80, 40), (33, 8)):
        run(3, 11, 4, 2, D, R, False, dtype, pad=pad, order=order, out_order=out_order)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pos", ["none", "any", "padding"])
def test_positions(pos, dtype):
    for D, R in ((128, 128), (64, 0), (90, 30)):
        run(2, 37, 6, 2, D, R, True, dtype, pos=pos)
        run(2, 37, 6, 2, D, R, False, dtype, pos=pos, weights=False, accumulate=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sides_that_are_left_out(dtype):
    run(2, 5, 4, 0, 64, 64, False, dtype)
    run(2, 5, 0, 3, 64, 64, False, dtype)
    run(2, 5, 0, 0, 64, 64, False, dtype)
    run(0, 5, 4, 2, 64, 64, False, dtype)
    run(2, 0, 4, 2, 64, 64, False, dtype, accumulate=True)


@pytest.mark.gpu
def test_sizes_of_values():
    """Rows far below eps, far above 1, and of zeros."""
    for scale in (0.0, 1e-30, 1e-3, 1e15):
        for D in (64, 50):
            run(1, 6, 3, 2, D, 32, False, "f32", scale=scale)
            run(1, 6, 3, 2, D, 32, True, "bf16", scale=scale)
    run(1, 6, 3, 2, 64, 32, False, "f32", scale=0.0, eps=2.0 ** -126)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_broken_rows_stay_alone(dtype):
    """A NaN or an infinity in a row, or in padding, reaches no other row; padding is zero whatever it holds."""
    r = np.random.default_rng(2)
    B, S, Hq, Hk = 1, 9, 4, 2
    for D, R in ((64, 64), (32, 32), (50, 10)):
        x = [r.standard_normal((B, S, H, D)) for H in (Hq, Hk)]
        clean = [y.copy() for y in x]
        x[0][0, 2, 1, 3], x[0][0, 4, :, :], x[1][0, 5, 0, 0] = np.nan, np.inf, -np.inf
        where = np.arange(S)
        where[4] = -1
        table = floats(rope_table(S, R))
        got = []
        for v in (x, clean):
            X = [Strided(y, dtype) for y in v]
            out, dX = ([Strided(0 * y, dtype) for y in clean] for _ in range(2))
            dg = [DB(4 * D) for _ in range(2)]
            a = (TYPE[dtype], B, S, Hq, Hk, D, R, False, EPS, ints(where), table, S, X[0], X[0].strides, X[1], X[1].strides,
                 None, None)
            hip.qk_norm_rope_fwd(*a, out[0], out[0].strides, out[1], out[1].strides)
            dY = [Strided(y, dtype) for y in clean]
            size = hip.qk_norm_rope_bwd_workspace(D)
            hip.qk_norm_rope_bwd(*a, TYPE[dtype], dY[0], dY[0].strides, dY[1], dY[1].strides, TYPE[dtype], dX[0], dX[0].strides,
                                 dX[1], dX[1].strides, *dg, False, DB(size), size)
            got.append([y.get() for y in out + dX])
        for i, (a, b) in enumerate(zip(*got)):
            bad = np.zeros(a.shape[:3], bool)
            bad[0, (2, 5)[i % 2], (1, 0)[i % 2]] = True
            assert np.isnan(a[bad]).any() and np.array_equal(a[~bad], b[~bad])
            assert (a[0, 4] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("Hq,Hk,D,R", [(6, 2, 64, 64), (20, 9, 128, 64), (3, 1, 50, 50), (2, 2, 300, 300)])
def test_padding_is_zero_whatever_the_rest_holds(Hq, Hk, D, R, dtype):
    """NaN in padding's rows, NaN and infinities in the table's first row and in the weights."""
    r = np.random.default_rng(3)
    B, S = 2, 5
    where = np.array([[-1, 1, 2, 9, -7], [3, -1, 9, 1, 2]])
    pad = (where < 0) | (where >= 4)
    table = rope_table(4, R)
    table[0, ::2], table[0, 1::2] = np.nan, np.inf
    x = [r.standard_normal((B, S, H, D)) for H in (Hq, Hk, Hq, Hk)]
    for v in x:
        v[pad] = np.nan
    Q, K, dQo, dKo = [Strided(v, dtype, (0, 1, 2), 0) for v in x]
    out = [Strided(np.full((B, S, H, D), 7.0), dtype, (0, 2, 1), 0) for H in (Hq, Hk, Hq, Hk)]
    for g in (np.inf, np.nan, 1.0):
        gb = [floats(np.full(D, g, np.float32)) for _ in range(2)]
        dg = [floats(np.zeros(D, np.float32)) for _ in range(2)]
        a = (TYPE[dtype], B, S, Hq, Hk, D, R, False, EPS, ints(where), floats(table), 4, Q, Q.strides, K, K.strides, *gb)
        hip.qk_norm_rope_fwd(*a, out[0], out[0].strides, out[1], out[1].strides)
        size = hip.qk_norm_rope_bwd_workspace(D)
        ws = DB(size)
        hip.qk_norm_rope_bwd(*a, TYPE[dtype], dQo, dQo.strides, dKo, dKo.strides, TYPE[dtype], out[2], out[2].strides, out[3],
                             out[3].strides, *dg, False, ws, size)
        for o in out:
            assert (o.get()[pad] == 0).all()
            assert g != 1.0 or np.isfinite(o.get()).all()
        for d in dg:   # the weights have no part in it
            assert np.isfinite(d.numpy()).all()


@pytest.mark.gpu
def test_many_rows_and_reruns():
    """More rows than waves: each wave takes several.  Reruns are equal bit for bit."""
    a = run(2, 1500, 7, 3, 64, 64, False, "bf16", "f32", "bf16")
    b = run(2, 1500, 7, 3, 64, 64, False, "bf16", "f32", "bf16")
    assert all(np.array_equal(x, y) for x, y in zip(a, b))
    run(1, 3001, 5, 1, 48, 20, True, "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("S,Hq,Hk,D,R", [(9001, 6, 2, 64, 64), (9001, 1, 1, 32, 16), (700, 40, 8, 32, 32), (9001, 3, 1, 30, 10),
                                         (2500, 1, 2, 128, 128)])
def test_units(S, Hq, Hk, D, R, dtype):
    """Whole tokens to a wave and parts of one, several tokens at once, waves that take several units; padded ends."""
    run(1, S, Hq, Hk, D, R, False, dtype, pos="any")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,pairs", [("f32", False), ("bf16", False), ("bf16", True)])
@pytest.mark.parametrize("shape", [(1, 9, 40, 9, 100, 50), (2, 3, 4, 1, 100, 100), (1, 7, 5, 9, 250, 250), (1, 5, 3, 7, 301, 50),
                                   (1, 4, 2, 5, 511, 510), (1, 5, 3, 2, 1001, 50), (1, 3, 5, 1, 1023, 1022)],
                         ids=lambda s: "x".join(map(str, s)))
def test_rows_in_no_whole_pieces(shape, dtype, pairs):
    run(*shape, pairs, dtype, grad="f32", pos="any", pad=1, seed=7)


@pytest.mark.gpu
@pytest.mark.parametrize("D,R", [(128, 128), (80, 40), (50, 10)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_in_place(dtype, D, R):
    """An output in its input's place gives what it gives apart."""
    r = np.random.default_rng(3)
    B, S, Hq, Hk = 2, 21, 6, 2
    table = floats(rope_table(S, R))
    X, Y = ([Strided(r.standard_normal((B, S, H, D)), dtype) for H in (Hq, Hk)] for _ in range(2))
    out, dX = ([Strided(np.zeros((B, S, H, D)), dtype) for H in (Hq, Hk)] for _ in range(2))
    ws, size = DB(hip.qk_norm_rope_bwd_workspace(D)), hip.qk_norm_rope_bwd_workspace(D)
    dt = TYPE[dtype]

    def fwd(to):
        hip.qk_norm_rope_fwd(dt, B, S, Hq, Hk, D, R, False, EPS, None, table, S, X[0], X[0].strides, X[1], X[1].strides, None,
                             None, to[0], to[0].strides, to[1], to[1].strides)

    def bwd(to):
        hip.qk_norm_rope_bwd(dt, B, S, Hq, Hk, D, R, False, EPS, None, table, S, X[0], X[0].strides, X[1], X[1].strides, None,
                             None, dt, Y[0], Y[0].strides, Y[1], Y[1].strides, dt, to[0], to[0].strides, to[1], to[1].strides,
                             None, None, False, ws, size)
    bwd(dX)
    want = [x.raw() for x in dX]
    bwd(Y)
    assert all(np.array_equal(x.raw(), w) for x, w in zip(Y, want))
    fwd(out)
    want = [x.raw() for x in out]
    fwd(X)
    assert all(np.array_equal(x.raw(), w) for x, w in zip(X, want))


@pytest.mark.gpu
def test_gradient_against_differences():
    """sum(w out) along a random direction of length 1: the difference over 2 h, h = 2^-5, is off by h^2 / 6 of the third
    derivative (|w|, |r| and |v| of order 1 to 8 a row, under 1e-2 of the result) and by the fp32 outputs' u
    |w . out| / h, under 1e-4."""
    r = np.random.default_rng(5)
    B, S, Hq, Hk, D, R, h = 1, 3, 2, 1, 64, 32, 2.0 ** -5
    table = floats(rope_table(S, R))
    g = [floats(1 + 0.3 * r.standard_normal(D)) for _ in range(2)]
    x = [r.standard_normal((B, S, H, D)) for H in (Hq, Hk)]
    w = [r.standard_normal((B, S, H, D)).astype(np.float32) for H in (Hq, Hk)]
    v = [r.standard_normal((B, S, H, D)) for H in (Hq, Hk)]
    norm = np.sqrt(sum((y * y).sum() for y in v))
    v = [y / norm for y in v]

    def args(x):
        X = [Strided(y, "f32") for y in x]
        return X, (hip.F32, B, S, Hq, Hk, D, R, False, EPS, None, table, S, X[0], X[0].strides, X[1], X[1].strides, *g)

    def f(x):
        X, a = args(x)
        out = [Strided(0 * y, "f32") for y in x]
        hip.qk_norm_rope_fwd(*a, out[0], out[0].strides, out[1], out[1].strides)
        return sum((o.get() * y).sum() for o, y in zip(out, w))

    X, a = args(x)
    dX, dY = [Strided(0 * y, "f32") for y in x], [Strided(y, "f32") for y in w]
    size = hip.qk_norm_rope_bwd_workspace(D)
    hip.qk_norm_rope_bwd(*a, hip.F32, dY[0], dY[0].strides, dY[1], dY[1].strides, hip.F32, dX[0], dX[0].strides, dX[1],
                         dX[1].strides, None, None, False, DB(size), size)
    slope = sum((d.get() * y).sum() for d, y in zip(dX, v))
    diff = (f([y + h * z for y, z in zip(x, v)]) - f([y - h * z for y, z in zip(x, v)])) / (2 * h)
    assert abs(slope - diff) <= 2e-2 * max(abs(slope), 0.1), (slope, diff)


@pytest.mark.gpu
@pytest.mark.parametrize("P,R,base", [(1, 2, 10000.0), (4097, 128, 10000.0), (131072, 64, 500000.0), (7, 2, 1.0)])
def test_table(P, R, base):
    """Angles in 64 bits: cosine and sine to one rounding, and what 2^17 radians lose in fp64 (2^17 2^-52 a few times)."""
    out = DB.empty((P, R), np.float32)
    hip.rope_table(P, R, base, out)
    a = np.arange(P)[:, None] * base ** (-2.0 * np.arange(R // 2) / R)
    within(out.numpy(), np.concatenate([np.cos(a), np.sin(a)], 1), U + 2.0 ** -30)
