"""Attention of one new token over a paged cache against plain formulas in 64 bits.

Tolerances (u = 2^-24, ub = 2^-8).  A score is a sum of D products in fp32 of operands that the types
hold exactly (8-bit values; a fp32 query as the kernel takes it, to 2^-24): random signs leave about sqrt(D) u of
scale sum |q k| = A, its scale, maximum and exponential's argument 8 u of it: dz = (2 sqrt(D) + 8) u A.
Every p is off by exp(dz): o by at most 2 dz of max |v|, lse by dz.  p has 16 bits or more where the
model's type is bf16 (2^-16 of max |v|), 24 where it is fp32; the sums over T tokens add up in 64 chains and
more: 64 u of max |v|.  Then one rounding to the output's type.
"""
import ctypes

import numpy as np
import pytest

from _decoder import TOP, TYPE, U, UB, Cache, Strided, attention, ints, rounded, within
from _gpu import DB
from dreamcompiler_amd import hip

KINDS = [("f32", "f32"), ("f32", "i8"), ("f32", "f8"), ("bf16", "bf16"), ("bf16", "i8"), ("bf16", "f8")]


class Case:
    def __init__(self, dtype, kind, lens, Hq, Hk, D, page, window=0, max_len=None, order=(0, 1), pad=0, seed=0, sharp=2.0,
                 spoil=(), change=None, lse=True, scale=None, ld=None):
        r = np.random.default_rng(seed)
        self.dtype, self.kind, self.lens, self.Hq, self.Hk, self.D = dtype, kind, lens, Hq, Hk, D
        B = len(lens)
        self.window, self.scale = window, scale or D ** -0.5
        self.c = c = Cache(kind, lens, Hk, D, page, seed, ld=ld)
        self.max_len = c.ld * page if max_len is None else max_len
        q = r.standard_normal((B, Hq, D)) * sharp
        kv = [[r.standard_normal((max(n, 0), Hk, D)) for n in lens] for _ in "KV"]
        if change:
            change(q, *kv)
        self.Q = Strided(q, dtype, order, pad)
        self.value = [[c.put(side, b, x) for b, x in enumerate(xs)] for side, xs in zip("KV", kv)]
        for b, i, v in spoil:
            c.table[b, i] = v
        c.upload()
        self.O = Strided(np.full((B, Hq, D), 7.0), dtype, order, pad)
        self.lse = DB.from_numpy(np.full((max(B, 1), Hq), 7.0, np.float32)) if lse else None
        self.size = hip.paged_attention_workspace(TYPE[kind], B, Hq, Hk, D, self.max_len)
        self.ws = DB(max(self.size, 16))

    def run(self):
        hip.paged_attention(TYPE[self.dtype], TYPE[self.kind], len(self.lens), self.Hq, self.Hk, self.D, self.scale,
                            self.window, self.Q, self.Q.strides, self.c.lbuf, self.max_len, *self.c.args(), self.O,
                            self.O.strides, self.lse, self.ws, self.size)
        return self

    def wipe(self):
        for b, n in ((self.O.buf, self.O.full.nbytes), (self.lse, 4 * len(self.lens) * self.Hq)):
            hip.check(hip.load().dh_memset(b.ptr, 0x55, n), "dh_memset")
        hip.sync()

    def values(self):
        return [self.O.raw(), self.lse.numpy()]

    def check(self):
        got, L = self.O.get(), self.lse.numpy() if self.lse else None
        c = self.c
        for b, n in enumerate(self.lens):
            n = min(max(n, 0), self.max_len)
            t = np.arange(max(n - self.window, 0) if self.window else 0, n)
            ids = c.table[b, t // c.page] if len(t) else t
            t = t[(ids >= 0) & (ids < c.pages)]
            K, V = (x[b][t] for x in self.value)
            o, lse, A = attention(self.Q.value[b], K, V, self.scale)
            big = np.abs(V).max() if V.size else 0.0
            dz = (2 * self.D ** 0.5 + 8) * U * A
            tol = ((2 * dz + 64 * U + (2.0 ** -16 if self.dtype == "bf16" else 0)) * big)[:, None]
            within(got[b], o, tol + (UB * (np.abs(o) + tol) if self.dtype == "bf16" else 0))
            if L is not None:
                within(L[b], lse, dz + 64 * U + 2 * U * np.abs(np.where(np.isfinite(lse), lse, 0)))
        return self


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("Hq,Hk,D,page", [(1, 1, 16, 16), (4, 2, 32, 16), (16, 16, 64, 32), (12, 3, 80, 16), (8, 1, 96, 64),
                                          (32, 8, 128, 16), (10, 2, 128, 128), (16, 1, 128, 256), (17, 1, 64, 16),
                                          (40, 2, 128, 32), (6, 6, 192, 16), (20, 1, 256, 64), (64, 1, 112, 4096),
                                          (33, 1, 48, 16)])
def test_heads_and_pages(Hq, Hk, D, page, dtype, kind):
    Case(dtype, kind, [1, 37, 0, 300], Hq, Hk, D, page).run().check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
def test_lengths(dtype, kind):
    """Around the ends of tiles, pages and chunks; empty ones and negative ones among them."""
    edge = [0, -7, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513, 767, 1023, 1024, 1025]
    Case(dtype, kind, edge, 8, 2, 64, 16).run().check()
    Case(dtype, kind, [3000, 1, 2049], 4, 4, 128, 32, seed=1).run().check()
    Case(dtype, kind, [20011], 8, 1, 128, 16, seed=2).run().check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("D", [32, 128, 192])
def test_long_chunks_of_many_sequences(D, dtype, kind):
    """Sequences enough for whole chunks: up to 2048 tokens, of more pages than lanes, by eight waves; and ones that
    are not split at all."""
    Hk = 1
    lens = [4100, 3000, 17, 0] + [1 + b % 40 for b in range(508)]
    chunk, splits, _, _ = hip.paged_attention_plan(TYPE[kind], len(lens), 2, Hk, D, 4112, 0)
    assert splits >= 2 and (D > 32 or chunk > 1024)
    Case(dtype, kind, lens, 2, Hk, D, 16).run().check()
    lens = [1088, 1087, 1025, 1024, 1000] + [3] * 123
    assert hip.paged_attention_plan(TYPE[kind], 128, 2, Hk, D, 1088, 0)[1] == 1
    Case(dtype, kind, lens, 2, Hk, D, 16).run().check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("D,T", [(32, 5000), (48, 9000), (96, 5000), (112, 9000), (160, 2500), (208, 1500), (256, 9000)])
def test_joins(D, T, dtype, kind):
    """Chunks for one, four and sixteen waves, of every length of a row."""
    Case(dtype, kind, [T, T // 2, 600, 5], 3, 1, D, 32).run().check()
    Case(dtype, kind, [T // 3, 129], 34, 2, D, 16, window=700).run().check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("window", [1, 2, 16, 31, 100, 257, 1000, 2 ** 31 - 1])
def test_windows(window, dtype, kind):
    Case(dtype, kind, [0, 1, 100, 258, 999, 1300], 6, 2, 64, 16, window=window).run().check()
    if window <= 257:
        Case(dtype, kind, [6001, 3000, 2], 4, 1, 128, 16, window=window).run().check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
def test_bounds_of_lengths(dtype, kind):
    """max_len below the lengths cuts them off; above, nothing changes; 0 leaves nothing."""
    lens = [600, 40, 0, 333]
    a = Case(dtype, kind, lens, 4, 2, 64, 16).run().check()
    b = Case(dtype, kind, lens, 4, 2, 64, 16, ld=8192).run().check()
    Case(dtype, kind, lens, 4, 2, 64, 16, max_len=100).run().check()
    Case(dtype, kind, lens, 4, 2, 64, 16, max_len=1).run().check()
    Case(dtype, kind, lens, 4, 2, 64, 16, max_len=0).run().check()
    assert a.max_len == 608 and b.max_len == 131072
    assert Case(dtype, kind, [], 4, 2, 64, 16).run() is not None


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
def test_pages_that_hold_nothing(dtype, kind):
    """Bad table entries: in the middle, first, last, all of a sequence's; far outside the pages."""
    far = [-1, 10 ** 6, 2 ** 31 - 1, -2 ** 31]
    Case(dtype, kind, [100, 64, 600, 33, 47], 8, 2, 64, 16,
         spoil=[(0, 2, far[0]), (0, 6, far[1])] + [(1, i, far[i]) for i in range(4)]
         + [(2, i, far[i % 4]) for i in range(0, 38, 3)] + [(3, 0, far[2]), (4, 2, far[3])]).run().check()
    Case(dtype, kind, [900], 4, 1, 128, 64, spoil=[(0, i, -1) for i in range(1, 12)]).run().check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
def test_shared_pages(dtype, kind):
    """A prefix that sequences share, and a page that one sequence has twice."""
    x = Case(dtype, kind, [700, 150, 64], 6, 2, 64, 16)
    for b in (1, 2):
        x.c.table[b, :4] = x.c.table[0, :4]
    x.c.table[1, 6] = x.c.table[1, 5]
    x.c.upload()
    for v in x.value:
        v[1][:64], v[2][:64] = v[0][:64], v[0][:64]
        v[1][96:112] = v[1][80:96]
    x.run().check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
def test_many_short_sequences(dtype, kind):
    Case(dtype, kind, [(5 * b) % 19 for b in range(3000)], 2, 1, 16, 16).run().check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("pad,order", [(0, (1, 0)), (3, (0, 1)), (8, (1, 0)), (1, (1, 0))])
def test_strides(pad, order, dtype, kind):
    Case(dtype, kind, [50, 7, 290], 6, 3, 80, 16, order=order, pad=pad).run().check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
def test_sharp_and_flat(dtype, kind):
    """One token with all the weight, scores hundreds apart, equal scores; the largest first and last."""
    def peak(at):
        def change(q, K, V):
            for b, k in enumerate(K):
                if len(k):
                    k[at if at >= 0 else len(k) - 1] = 5 * q[b, :1]
        return change

    def flat(q, K, V):
        q[:] = 0

    for change in (peak(0), peak(-1), peak(20), flat):
        Case(dtype, kind, [700, 21, 64], 4, 1, 64, 16, change=change).run().check()
    Case(dtype, kind, [700, 21, 64], 4, 1, 64, 16, sharp=30.0).run().check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", [("f32", "f32"), ("bf16", "bf16")])
def test_infinities(dtype, kind):
    """A key that no query wants (scores of -infinity) counts for nothing; where there is no other, as an
    empty row; a NaN that is seen stays in its head."""
    def away(q, K, V):
        q[:] = np.abs(q)
        for k in K:
            k[::2] = -np.inf
        K[1][:] = -np.inf

    x = Case(dtype, kind, [333, 40, 64], 4, 2, 64, 16, change=away).run()
    got, L = x.O.get(), x.lse.numpy()
    assert (got[1] == 0).all() and (L[1] == -np.inf).all()
    for b in (0, 2):
        o, lse, A = attention(x.Q.value[b], x.value[0][b][1::2], x.value[1][b][1::2], x.scale)
        within(got[b], o, 1e-4 + UB * np.abs(o))
        within(L[b], lse, 1e-4)

    def one(q, K, V):
        K[0][5, 1] = np.nan

    x = Case(dtype, kind, [70, 70], 4, 2, 64, 16, change=one).run()
    got = x.O.get()
    assert np.isnan(got[0, 2:]).all() and np.isfinite(got[0, :2]).all() and np.isfinite(got[1]).all()


@pytest.mark.gpu
def test_without_lse_and_reruns():
    for dtype, kind in KINDS:
        x = Case(dtype, kind, [1500, 20], 8, 2, 128, 16, lse=False).run().check()
        a = x.O.raw()
        x.run()
        assert np.array_equal(a, x.O.raw())


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Pages whose offsets pass 2^32 values."""
    Hq, Hk, D, page, pages = 16, 8, 256, 4096, 700
    Kc, Vc = DB(pages * Hk * page * D), DB(pages * Hk * page * D)
    Ks, Vs = (DB(pages * Hk * page * 4) for _ in "KV")
    r = np.random.default_rng(0)
    held = (pages, page, ints([[699]]), 1, Kc, Vc, Ks, Vs)
    T = 50
    K, V = (Strided(r.standard_normal((T, Hk, D)), "bf16") for _ in "KV")
    Q, O = Strided(r.standard_normal((1, Hq, D)), "bf16"), Strided(np.zeros((1, Hq, D)), "bf16")
    n = ints([T])
    hip.kv_cache_write(hip.BF16, hip.F8, 1, T, Hk, D, K, K.strides, V, V.strides, ints([0, T]), n, *held)
    back = [Strided(np.zeros((T, Hk, D)), "f32") for _ in "KV"]
    hip.kv_cache_read(hip.F32, hip.F8, 1, T, Hk, D, back[0], back[0].strides, back[1], back[1].strides, ints([0, T]), n, *held)
    size = hip.paged_attention_workspace(hip.F8, 1, Hq, Hk, D, page)
    hip.paged_attention(hip.BF16, hip.F8, 1, Hq, Hk, D, D ** -0.5, 0, Q, Q.strides, n, page, *held, O, O.strides, None,
                        DB(max(size, 16)), size)
    o, _, A = attention(Q.value[0], back[0].get(), back[1].get(), D ** -0.5)
    within(O.get()[0], o, 2.0 ** -15 * 4 + UB * np.abs(o))
