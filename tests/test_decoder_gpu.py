"""A decoder's attention as it is used: training (norm and rotation, flash attention, their gradients) and
serving (norm and rotation, the cache, attention of the new token), against plain formulas in 64 bits; and
the calls recorded into graphs that run at once.

Tolerances.  Training in fp32: each stage is held to 64 u = 4e-6 of its terms in its own tests; through scores
of size |q k| scale <= 30 an error of 2e-5 in p and so in the gradients' terms: 1e-4 of the largest value.
Serving: keys and values are what the cache's type makes of what the norm gave, read back from it, so what is
left is the attention's own error and one rounding (fp32 1e-5, bf16 2^-8 and 2^-15 of the largest value).
"""
import ctypes

import numpy as np
import pytest

from _decoder import TOP, TYPE, U, UB, Cache, Strided, attention, floats, ints, norm_rope, rope_table, within
from _gpu import DB
from dreamcompiler_amd import hip

EPS = 1e-6


def causal(Q, K, V, scale, dO):
    """B x H x S x D in fp64: O and its gradients."""
    S = Q.shape[2]
    z = scale * Q @ K.transpose(0, 1, 3, 2)
    z = np.where(np.tril(np.ones((S, S), bool)), z, -np.inf)
    p = np.exp(z - z.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    dp = dO @ V.transpose(0, 1, 3, 2)
    dz = p * (dp - (dp * p).sum(-1, keepdims=True)) * scale
    return p @ V, dz @ K, dz.transpose(0, 1, 3, 2) @ Q, p.transpose(0, 1, 3, 2) @ dO


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,H,D,R,pairs", [(2, 70, 3, 64, 64, False), (1, 129, 2, 128, 64, True), (2, 33, 4, 32, 16, False)])
def test_training(B, S, H, D, R, pairs):
    """From the projections' rows to gradients of queries, keys, values and the norm's weights."""
    r = np.random.default_rng(1)
    x = r.standard_normal((B, S, 3 * H, D)).astype(np.float32)
    X = DB.from_numpy(x)
    row = 3 * H * D
    wide, slices = (S * row, row, D), (H * S * D, D, S * D)
    table, g = rope_table(S, R), 1 + 0.2 * r.standard_normal((2, D)).astype(np.float32)
    tb, gb = floats(table), [floats(y) for y in g]
    dO = r.standard_normal((B, H, S, D)).astype(np.float32)
    Q, K, O, dQ, dK, dV = (DB(4 * B * H * S * D) for _ in range(6))
    V = DB.from_numpy(np.ascontiguousarray(x[:, :, 2 * H:].transpose(0, 2, 1, 3)))
    lse, dX = DB(4 * B * H * S), DB.from_numpy(np.zeros_like(x))
    dg = [DB(4 * D) for _ in range(2)]
    size = hip.qk_norm_rope_bwd_workspace(D)
    a = (hip.F32, B, S, H, H, D, R, pairs, EPS, None, tb, S, X.ptr, wide, X.ptr + 4 * H * D, wide, *gb)
    scale = D ** -0.5
    hip.qk_norm_rope_fwd(*a, Q, slices, K, slices)
    hip.flash_fwd(hip.F32, B * H, S, D, scale, True, Q, K, V, O, lse)
    dOb = DB.from_numpy(dO)
    hip.flash_bwd(hip.F32, B * H, S, D, scale, True, Q, K, V, O, dOb, lse, dQ, dK, dV, 0)
    hip.qk_norm_rope_bwd(*a, hip.F32, dQ, slices, dK, slices, hip.F32, dX.ptr, wide, dX.ptr + 4 * H * D, wide, *dg, False,
                         DB(size), size)
    x = x.astype(np.float64)
    pos = np.tile(np.arange(S), (B, 1))
    q, k, v = x[:, :, :H], x[:, :, H:2 * H], x[:, :, 2 * H:].transpose(0, 2, 1, 3)
    Qr, Kr = (norm_rope(y, w.astype(np.float64), pos, table, R, pairs, EPS).transpose(0, 2, 1, 3) for y, w in zip((q, k), g))
    Or, dQr, dKr, dVr = causal(Qr, Kr, v, scale, dO.astype(np.float64))
    shape = (B, H, S, D)
    got = dX.numpy((B, S, 3 * H, D), np.float32)
    for y, ref in ((O.numpy(shape, np.float32), Or), (dV.numpy(shape, np.float32), dVr)):
        within(y, ref, 1e-4 * np.abs(ref).max())
    for i, (y, d) in enumerate(((q, dQr), (k, dKr))):
        dx, dw, _, terms = norm_rope(y, g[i].astype(np.float64), pos, table, R, pairs, EPS, d.transpose(0, 2, 1, 3))
        within(got[:, :, i * H:(i + 1) * H], dx, 1e-4 * np.abs(dx).max())
        within(dg[i].numpy((D,), np.float32), dw, 1e-4 * np.abs(dw).max() + 1e-5 * terms.max())
    assert (got[:, :, 2 * H:] == 0).all()


class Server:
    """Sequences that go on token by token: a prompt, then single tokens, through one cache."""

    def __init__(self, dtype, kind, Hq, Hk, D, page, prompts, steps, seed=0):
        r = np.random.default_rng(seed)
        self.dt, self.dtype, self.kind, self.Hq, self.Hk, self.D = TYPE[dtype], dtype, kind, Hq, Hk, D
        self.B, self.prompts, self.steps = len(prompts), prompts, steps
        self.cache = Cache(kind, [n + steps for n in prompts], Hk, D, page, seed)
        self.cache.upload()
        self.P = max(prompts) + steps
        self.table = floats(rope_table(self.P, D))
        self.g = [floats(1 + 0.2 * r.standard_normal(D)) for _ in range(2)]
        self.max_len = self.cache.ld * page
        self.size = hip.paged_attention_workspace(TYPE[kind], self.B, Hq, Hk, D, self.max_len)
        self.ws = DB(max(self.size, 16))
        self.r = r

    def tokens(self, counts, lens):
        """The projections' rows of counts[b] new tokens of each sequence, and what their calls need."""
        n, heads = sum(counts), self.Hq + 2 * self.Hk
        first = np.concatenate([[0], np.cumsum(counts)])
        pos = np.concatenate([np.arange(l - c, l) for c, l in zip(counts, lens)])
        X = Strided(self.r.standard_normal((1, n, heads * self.D)), self.dtype)
        q, k = Strided(np.zeros((1, n, self.Hq, self.D)), self.dtype), Strided(np.zeros((1, n, self.Hk, self.D)), self.dtype)
        return dict(n=n, X=X, q=q, k=k, pos=ints(pos), first=ints(first), len=ints(lens), row=heads * self.D)

    def write(self, t):
        D, Hq, Hk, e, row = self.D, self.Hq, self.Hk, 4 if self.dtype == "f32" else 2, t["row"]
        x, wide = t["X"].ptr, (t["n"] * row, row, D)
        hip.qk_norm_rope_fwd(self.dt, 1, t["n"], Hq, Hk, D, D, False, EPS, t["pos"], self.table, self.P, x, wide,
                             x + e * Hq * D, wide, *self.g, t["q"], t["q"].strides, t["k"], t["k"].strides)
        hip.kv_cache_write(self.dt, TYPE[self.kind], self.B, t["n"], Hk, D, t["k"], t["k"].strides[1:],
                           x + e * (Hq + Hk) * D, (row, D), t["first"], t["len"], *self.cache.args())

    def attend(self, t, O, lse):
        hip.paged_attention(self.dt, TYPE[self.kind], self.B, self.Hq, self.Hk, self.D, self.D ** -0.5, 0, t["q"],
                            t["q"].strides[1:], t["len"], self.max_len, *self.cache.args(), O, O.strides, lse, self.ws, self.size)


KINDS = [("f32", "f32"), ("f32", "i8"), ("bf16", "bf16"), ("bf16", "i8"), ("bf16", "f8")]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("Hq,Hk,D,page", [(4, 2, 64, 16), (8, 1, 128, 32), (3, 3, 80, 64)])
def test_serving(Hq, Hk, D, page, dtype, kind):
    s = Server(dtype, kind, Hq, Hk, D, page, [15, 1, 100, 33], 3)
    s.write(s.tokens(s.prompts, s.prompts))
    for step in range(1, s.steps + 1):
        lens = [n + step for n in s.prompts]
        t = s.tokens([1] * s.B, lens)
        s.write(t)
        O, lse = Strided(np.zeros((s.B, Hq, D)), dtype), DB(4 * s.B * Hq)
        s.attend(t, O, lse)
        # the whole context, read back
        first = np.concatenate([[0], np.cumsum(lens)])
        n = int(first[-1])
        KV = [Strided(np.zeros((n, Hk, D)), "f32" if kind in TOP else dtype) for _ in "KV"]
        hip.kv_cache_read(TYPE[KV[0].dtype] if kind in TOP else s.dt, TYPE[kind], s.B, n, Hk, D, KV[0], KV[0].strides, KV[1],
                          KV[1].strides, ints(first), t["len"], *s.cache.args())
        K, V = (x.get() for x in KV)
        q = t["q"].get()[0]
        # the new token's key is what the norm gave, to the cache's type
        new = t["k"].get()[0]
        for b in range(s.B):
            top = np.abs(new[b]).max(-1, keepdims=True)
            off = {"f32": 0, "bf16": 0, "i8": 0.51 / 127 * top, "f8": 2.0 ** -4 * np.abs(new[b]) + 2.0 ** -10 * top / 448}[kind]
            within(K[first[b + 1] - 1], new[b], off)
            o, L, A = attention(q[b], K[first[b]:first[b + 1]], V[first[b]:first[b + 1]], D ** -0.5)
            tol = (1e-5 if dtype == "f32" else 2.0 ** -15) * np.abs(V).max()
            within(O.get()[b], o, tol + (UB * np.abs(o) if dtype == "bf16" else 0))
            within(lse.numpy((s.B, Hq), np.float32)[b], L, 1e-5 * (1 + np.abs(L)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", [("f32", "f32"), ("bf16", "bf16")])
def test_prompt_by_flash_and_by_steps(dtype, kind):
    """The last row of causal flash attention over a prompt is what attention of its last token over the cache gives:
    both to one rounding of the output, fp32 4e-6 and bf16 2^-8 of the value and, as flash rounds its p, of the largest."""
    S, H, D = 150, 4, 64
    s = Server(dtype, kind, H, H, D, 16, [S], 0, seed=4)
    t = s.tokens([S], [S])
    s.write(t)
    e = 4 if dtype == "f32" else 2
    Q, K, V, O = (Strided(np.zeros((H, S, D)), dtype) for _ in range(4))
    x = t["X"].get()[0].reshape(S, 3 * H, D)
    V = Strided(x[:, 2 * H:].transpose(1, 0, 2), dtype)
    wide, slices = (S * t["row"], t["row"], D), (H * S * D, D, S * D)
    hip.qk_norm_rope_fwd(s.dt, 1, S, H, H, D, D, False, EPS, t["pos"], s.table, s.P, t["X"].ptr, wide, t["X"].ptr + e * H * D,
                         wide, *s.g, Q, slices, K, slices)
    hip.flash_fwd(s.dt, H, S, D, D ** -0.5, True, Q, K, V, O, DB(4 * H * S))
    one = Strided(np.zeros((1, H, D)), dtype)
    last = t["q"].ptr + (S - 1) * H * D * e
    hip.paged_attention(s.dt, TYPE[kind], 1, H, H, D, D ** -0.5, 0, last, (H * D, D), t["len"], s.max_len, *s.cache.args(), one,
                        one.strides, None, s.ws, s.size)
    a, b = O.get()[:, -1], one.get()[0]
    within(a, b, 1e-5 if dtype == "f32" else 2 * UB * np.abs(b) + 2 * UB * np.abs(b).max())


def _runtime():
    R, v, p = ctypes.CDLL("libamdhip64.so"), ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p)
    for name, args in (("hipStreamCreate", [p]), ("hipStreamSynchronize", [v]), ("hipStreamDestroy", [v]),
                       ("hipStreamBeginCapture", [v, ctypes.c_int]), ("hipStreamEndCapture", [v, p]),
                       ("hipGraphInstantiate", [p, v, v, v, ctypes.c_size_t]), ("hipGraphLaunch", [v, v]),
                       ("hipGraphExecDestroy", [v]), ("hipGraphDestroy", [v])):
        getattr(R, name).argtypes = args
        getattr(R, name).restype = ctypes.c_int
    return R


class Step:
    """A serving step, and a gradient of the norm, whose calls can be recorded."""

    def __init__(self, dtype, kind, seed):
        self.s = s = Server(dtype, kind, 8, 2, 64, 16, [700, 33], 1, seed)
        s.write(s.tokens(s.prompts, s.prompts))
        self.t = s.tokens([1, 1], [701, 34])
        self.O, self.lse = Strided(np.zeros((2, 8, 64)), dtype), DB(4 * 16)
        r = np.random.default_rng(seed)
        self.dY = [Strided(r.standard_normal((1, 2, H, 64)), dtype) for H in (8, 2)]
        self.dX = [Strided(np.zeros((1, 2, H, 64)), dtype) for H in (8, 2)]
        self.dg = [DB(4 * 64) for _ in range(2)]
        self.size = hip.qk_norm_rope_bwd_workspace(64)
        self.ws = DB(self.size)
        hip.sync()

    def run(self):
        s, t = self.s, self.t
        s.write(t)
        s.attend(t, self.O, self.lse)
        e = 4 if s.dtype == "f32" else 2
        wide = (2 * t["row"], t["row"], 64)
        hip.qk_norm_rope_bwd(s.dt, 1, 2, 8, 2, 64, 64, False, EPS, t["pos"], s.table, s.P, t["X"].ptr, wide, t["X"].ptr + e * 8 * 64,
                             wide, *s.g, s.dt, self.dY[0], self.dY[0].strides, self.dY[1], self.dY[1].strides, s.dt, self.dX[0],
                             self.dX[0].strides, self.dX[1], self.dX[1].strides, *self.dg, False, self.ws, self.size)

    def wipe(self):
        for b, n in [(x.buf, x.full.nbytes) for x in [self.O, self.t["q"], self.t["k"], *self.dX]] + [(self.lse, 64)] + [
                (b, 256) for b in self.dg]:
            hip.check(hip.load().dh_memset(b.ptr, 0x55, n), "dh_memset")
        hip.sync()

    def values(self):
        hip.sync()
        return [x.raw() for x in [self.O, self.t["q"], self.t["k"], *self.dX]] + [self.lse.numpy((16,), np.float32)] + [
            b.numpy((64,), np.float32) for b in self.dg]


@pytest.mark.gpu
@pytest.mark.parametrize("a,b", [(("bf16", "bf16"), ("bf16", "f8")), (("f32", "f32"), ("f32", "i8"))])
def test_graphs_on_other_streams(a, b):
    """Recorded with nothing allocated, on streams of the caller's; two graphs replayed at once, three times, their
    results wiped between: what the library's own stream gives, bit for bit."""
    jobs = [Step(*a, seed=1), Step(*b, seed=2)]
    want = []
    for j in jobs:
        j.run()
        want.append(j.values())
    R, lib = _runtime(), hip.load()
    streams, graphs, exes = ([ctypes.c_void_p() for _ in jobs] for _ in range(3))
    ref = ctypes.byref
    try:
        for j, w, s, g, x in zip(jobs, want, streams, graphs, exes):
            assert R.hipStreamCreate(ref(s)) == 0
            hip.check(lib.dh_set_stream(s), "dh_set_stream")
            j.wipe()
            j.run()
            assert all(np.array_equal(v, u) for v, u in zip(j.values(), w))
            assert R.hipStreamBeginCapture(s, 0) == 0
            try:
                j.run()
            finally:
                end = R.hipStreamEndCapture(s, ref(g))
            assert end == 0 and R.hipGraphInstantiate(ref(x), g, None, None, 0) == 0
        lib.dh_set_stream(None)
        for _ in range(3):
            for j in jobs:
                j.wipe()
            for x, s in zip(exes, streams):
                assert R.hipGraphLaunch(x, s) == 0
            for s in streams:
                assert R.hipStreamSynchronize(s) == 0
            for j, w in zip(jobs, want):
                assert all(np.array_equal(v, u) for v, u in zip(j.values(), w))
            jobs[0].run()
            hip.sync()
    finally:
        lib.dh_set_stream(None)
        for s, g, x in zip(streams, graphs, exes):
            if x.value:
                R.hipGraphExecDestroy(x)
            if g.value:
                R.hipGraphDestroy(g)
            if s.value:
                R.hipStreamSynchronize(s)
                R.hipStreamDestroy(s)
