"""The operators around a decoder's attention where their sizes, addresses and values are at an edge: scores and values
that are not finite, single heads of very many tokens, thousands of sequences, rows at odd addresses, calls that need no
workspace.  Tolerances are those of the operators' own tests."""
import numpy as np
import pytest

from _decoder import (TOP, TYPE, U, UB, Cache, Strided, attention, decode, ints, norm_rope, quantised, rope_table,
                      rounded, within)
from _gpu import DB
from dreamcompiler_amd import hip
from test_kv_cache_gpu import read_back
from test_kv_cache_gpu import run as run_cache
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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
def test_attention_at_odd_addresses(dtype, kind):
    """Queries and results one value behind 16 bytes, lengths, table and lse four bytes."""
    x = Case(dtype, kind, [50, 1000, 290], 6, 3, 80, 16).run().check()
    want = x.values()
    e = 4 if dtype == "f32" else 2
    n = x.Q.full.size
    raw = x.Q.full.reshape(-1)
    Q, O = DB.from_numpy(np.concatenate([raw[:1], raw])), DB.from_numpy(np.concatenate([raw[:1], 0 * raw, raw[:1]]))
    len_, table = ints(np.concatenate([[9], x.c.lens])), ints(np.concatenate([[9], x.c.table.reshape(-1)]))
    lse = DB.from_numpy(np.full(3 * 6 + 2, 7.0, np.float32))
    a = x.c.args()
    hip.paged_attention(TYPE[dtype], TYPE[kind], 3, 6, 3, 80, x.scale, 0, Q.ptr + e, x.Q.strides, len_.ptr + 4, x.max_len,
                        a[0], a[1], table.ptr + 4, *a[3:], O.ptr + e, x.O.strides, lse.ptr + 4, x.ws, x.size)
    out = O.numpy((n + 2,), raw.dtype)
    assert np.array_equal(out[1:-1], want[0].reshape(-1)) and np.array_equal(out[[0, -1]], raw[[0, 0]])
    out = lse.numpy()
    assert np.array_equal(out[1:-1], want[1].reshape(-1)) and out[0] == out[-1] == 7.0


# ------------------------------------------------------------------------------ the cache

@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("pad", [1, 3])
def test_many_tokens_in_rows_of_no_whole_pieces(pad, dtype, kind):
    """A wave a row: more rows than waves of a launch, and more sequences than lanes."""
    run_cache(dtype, kind, [2100, 1, 900], [2100, 1, 450], 6, 32, 32, pad=pad)
    lens = [(7 * b) % 23 for b in range(150)]
    run_cache(dtype, kind, lens, [n if b % 3 else n // 2 for b, n in enumerate(lens)], 2, 48, 16, pad=pad)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", [("f32", "f8"), ("bf16", "bf16"), ("bf16", "i8")])
@pytest.mark.parametrize("pad", [0, 1])
def test_thousands_of_sequences(pad, dtype, kind):
    """More than 64 x 64 beginnings: three rounds of the search by 64."""
    lens = [(5 * b) % 4 for b in range(4500)]
    run_cache(dtype, kind, lens, [n if b % 3 else n // 2 for b, n in enumerate(lens)], 1, 16, 16, pad=pad)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", [("f32", "i8"), ("bf16", "bf16"), ("bf16", "f8")])
@pytest.mark.parametrize("Hk,T", [(1, 900000), (2, 450000), (3, 250000)])
def test_rounds_of_several_tokens(Hk, T, dtype, kind):
    """So many tokens that a wave makes more than one round over its own, with 16, 8 and 4 of them at once."""
    D, page = 16, 256
    r = np.random.default_rng(6)
    c = Cache(kind, [T], Hk, D, page).upload()
    K, V = (Strided(r.standard_normal((T, Hk, D)).astype(np.float32), dtype) for _ in "KV")
    first = ints([0, T])
    hip.kv_cache_write(TYPE[dtype], TYPE[kind], 1, T, Hk, D, K, K.strides, V, V.strides, first, c.lbuf, *c.args())
    out = [Strided(np.zeros((T, Hk, D), np.float32), dtype) for _ in "KV"]
    hip.kv_cache_read(TYPE[dtype], TYPE[kind], 1, T, Hk, D, out[0], out[0].strides, out[1], out[1].strides, first, c.lbuf,
                      *c.args())
    raw, scale = c.download()
    t = np.arange(T)
    at = (c.table[0, t // page], slice(None), t % page)
    for n, x, o in (("K", K, out[0]), ("V", V, out[1])):
        if kind in TOP:
            codes, s = quantised(x.value, kind)
            assert np.array_equal(decode(raw[n][at], kind), codes) and np.array_equal(scale[n][at], s)
        else:
            codes, s = x.value, None
            assert np.array_equal(raw[n][at], rounded(x.value, kind)[0])
        assert np.array_equal(o.get(), read_back(codes, s, kind, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [0, 1])
@pytest.mark.parametrize("first", [[5, 3, 9, 9], [-7, 4, 2, 12], [0, 2 ** 31 - 1, 3, 6], [0, 0, 0, 0], [9, 9, 9, 9]])
def test_beginnings_that_do_not_rise_keep_to_their_places(first, pad):
    """What no caller means: keys and values in buffers of their own, each told from the other, nothing read or written
    out of place, and rows of no sequence stay."""
    Hk, D, N = 2, 32, 8
    c = Cache("bf16", [20, 20, 20], Hk, D, 16).upload()
    K, V = (Strided(np.full((N, Hk, D), v), "bf16", pad=pad) for v in (1.0, -2.0))
    hip.kv_cache_write(hip.BF16, hip.BF16, 3, N, Hk, D, K, K.strides, V, V.strides, ints(first), c.lbuf, *c.args())
    out = [Strided(np.full((N, Hk, D), v), "bf16", pad=pad) for v in (7.0, 9.0)]
    hip.kv_cache_read(hip.BF16, hip.BF16, 3, N, Hk, D, out[0], out[0].strides, out[1], out[1].strides, ints(first), c.lbuf,
                      *c.args())
    raw = c.download()[0]
    nan, one, two = 0x7FC0, 0x3F80, 0xC000
    for n, o, v, bits, stays in (("K", out[0], 1.0, one, 7.0), ("V", out[1], -2.0, two, 9.0)):
        got = o.get()
        assert (np.isnan(got) | (got == 0) | (got == v) | (got == stays)).all()
        assert ((raw[n] == nan) | (raw[n] == bits)).all()
        if first in ([0, 0, 0, 0], [9, 9, 9, 9]):
            assert (got == stays).all() and (raw[n] == nan).all()


# ------------------------------------------------------------------------------ norm and rotation

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,R,shift", [(64, 64, 0), (64, 64, 1), (128, 64, 4), (50, 10, 1)])
def test_norm_at_odd_addresses(D, R, shift, dtype):
    """Rows `shift` values behind 16 bytes; weights, their gradients, table and positions four bytes behind them."""
    B, S, Hq, Hk, e = 2, 9, 6, 2, 4 if dtype == "f32" else 2
    r = np.random.default_rng(8)
    table, g = rope_table(S, R), 1 + 0.3 * r.standard_normal((2, D)).astype(np.float32)
    where = np.tile(np.arange(S), (B, 1))
    where[1, -2:] = -1
    lead = lambda x, t: DB.from_numpy(np.concatenate([np.zeros(1, t), np.asarray(x, t).reshape(-1)]))  # noqa: E731
    pos, tb, gb = lead(where, np.int32), lead(table, np.float32), [lead(y, np.float32) for y in g]

    def rows(H, fill=None):
        x = r.standard_normal((B, S, H, D)) if fill is None else np.full((B, S, H, D), fill)
        raw, value = rounded(x, dtype)
        return DB.from_numpy(np.concatenate([np.zeros(shift, raw.dtype), raw.reshape(-1)])), value

    X, Y, out, dX = ([rows(H, f) for H in (Hq, Hk)] for f in (None, None, 7.0, 7.0))
    st = [(S * H * D, H * D, D) for H in (Hq, Hk)]
    at = lambda t, i: t[i][0].ptr + shift * e  # noqa: E731
    dg = [lead(np.zeros(D), np.float32) for _ in range(2)]
    dt = TYPE[dtype]
    a = (dt, B, S, Hq, Hk, D, R, False, 1e-6, pos.ptr + 4, tb.ptr + 4, S, at(X, 0), st[0], at(X, 1), st[1], gb[0].ptr + 4,
         gb[1].ptr + 4)
    hip.qk_norm_rope_fwd(*a, at(out, 0), st[0], at(out, 1), st[1])
    size = hip.qk_norm_rope_bwd_workspace(D)
    hip.qk_norm_rope_bwd(*a, dt, at(Y, 0), st[0], at(Y, 1), st[1], dt, at(dX, 0), st[0], at(dX, 1), st[1], dg[0].ptr + 4,
                         dg[1].ptr + 4, False, DB(size), size)

    def got(t, i):
        H = (Hq, Hk)[i]
        raw = t[i][0].numpy((shift + B * S * H * D,), np.float32 if e == 4 else np.uint16)[shift:].reshape(B, S, H, D)
        return (raw if e == 4 else (raw.astype(np.uint32) << 16).view(np.float32)).astype(np.float64)

    for i in range(2):
        w = g[i].astype(np.float64)
        ref = norm_rope(X[i][1], w, where, table, R, False, 1e-6)
        flat = norm_rope(X[i][1], w, where * 0, table[:1] * 0 + 1, 0, False, 1e-6)
        within(got(out, i), ref, 48 * U * np.abs(flat).max(-1, keepdims=True) + (UB * np.abs(ref) * (1 + UB) if e == 2 else 0))
        dx, dw, by, terms = norm_rope(X[i][1], w, where, table, R, False, 1e-6, Y[i][1])
        within(got(dX, i), dx, 64 * U * by + (UB * (np.abs(dx) + 64 * U * by) if e == 2 else 0))
        d = dg[i].numpy((D + 1,), np.float32)
        assert d[0] == 0
        within(d[1:], dw, (64 + B * S * (Hq, Hk)[i]) * U * terms)
