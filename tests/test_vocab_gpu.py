"""Embedding, linear cross entropy and linear distillation against plain formulas in 64 bits.

Tolerances (u = 2^-24, the largest relative error of one fp32 rounding; ub = 2^-8 of one to bf16).
A product of length D with operands rounded to their type before the call is exact up to its fp32
sum, whose error is at most about sqrt(D) u of |h| |w| for operands of random sign; an fp32 operand
is taken to 2^-23 of itself or 2^-51 of its row's largest value.  With
|z| up to about 20 that gives logits to 1e-5, and as d exp(z) = exp(z) dz every probability to 1e-5
of itself; sums of them keep that.  So fp32 results are held to 2e-5 of the largest value of the
result (for the loss: of its largest, at least 1).  bf16 gradients: one rounding of G (ub of
each term of a sum, in random directions) and one of the result (ub of it): 2 ub = 2^-7 of the
result's largest value; the embedding's bf16 results are rounded once: ub.
"""
import ctypes

import numpy as np
import pytest

from _gpu import DB, bf16_bits, bits_to_f32
from dreamcompiler_amd import hip

F32_TOL, BF16_TOL, BF16_ONCE = 2e-5, 2.0 ** -7, 2.0 ** -8
DT = {"f32": hip.F32, "bf16": hip.BF16}


def store(x, dtype, ld=None):
    """x (R x C) on the device as `dtype` in rows of ld values (NaN between them), and its values."""
    x = np.asarray(x, np.float32)
    if dtype == "bf16":
        bits = bf16_bits(x)
        x = bits_to_f32(bits)
    ld = ld or x.shape[1]
    full = np.full((x.shape[0], ld), np.nan, np.float32)
    full[:, :x.shape[1]] = x
    raw = np.full((x.shape[0], ld), 0x7FC0, np.uint16) if dtype == "bf16" else full
    if dtype == "bf16":
        raw[:, :x.shape[1]] = bits
    return DB.from_numpy(raw), x.astype(np.float64)


def fetch(buf, shape, dtype, ld=None):
    ld = ld or shape[1]
    raw = buf.numpy((shape[0], ld), np.uint16 if dtype == "bf16" else np.float32)
    x = bits_to_f32(raw) if dtype == "bf16" else raw
    return x[:, :shape[1]].astype(np.float64), raw


def ints(x):
    return DB.from_numpy(np.asarray(x, np.int32))


def close(got, ref, tol, floor=0.0):
    scale = max(np.abs(ref).max(initial=0.0), floor)
    err = np.abs(got - ref).max(initial=0.0)
    assert np.isfinite(got).all() and err <= tol * scale, (err, tol * scale)


# ------------------------------------------------------------------------------ embedding

def emb_ref(ids, W, dY, scale):
    V = W.shape[0]
    ok = (ids >= 0) & (ids < V)
    Y = np.zeros((len(ids), W.shape[1]))
    Y[ok] = scale * W[ids[ok]]
    dW = np.zeros_like(W)
    np.add.at(dW, ids[ok], scale * dY[ok])
    return Y, dW


def run_embedding(ids, V, D, dtype, grad, ldx=0, accumulate=False, scale=1.5, seed=0):
    r = np.random.default_rng(seed)
    ids = np.asarray(ids, np.int32)
    N = len(ids)
    dW_, W = store(r.standard_normal((V, D)), dtype, D + ldx)
    dYb, dY = store(r.standard_normal((max(N, 1), D)), dtype, D + ldx)
    dY = dY[:N]
    Yb, _ = store(np.zeros((max(N, 1), D)), dtype, D + ldx)
    old = r.standard_normal((V, D)) if accumulate else np.full((V, D), np.nan)
    gb, old = store(old, grad, D + ldx)
    ib = ints(ids if N else [0])
    hip.embedding_fwd(DT[dtype], N, V, D, scale, ib, dW_, D + ldx, Yb, D + ldx)
    size = hip.embedding_bwd_workspace(N, V, D)
    assert size <= (N + 16) * (D + 511) // 2 + 18 * N + V + 16384
    ws = DB(max(size, 16))
    hip.embedding_bwd(DT[dtype], N, V, D, scale, ib, dYb, D + ldx, gb, D + ldx, DT[grad], accumulate,
                      ws, size)
    Y, rawY = fetch(Yb, (max(N, 1), D), dtype, D + ldx)
    G, rawG = fetch(gb, (V, D), grad, D + ldx)
    if ldx:   # what lies between the rows stays as it was
        for raw, t in ((rawY, dtype), (rawG, grad)):
            gap = raw[:, D:]
            assert (gap == 0x7FC0).all() if t == "bf16" else np.isnan(gap).all()
    refY, refG = emb_ref(ids, W, dY, scale)
    close(Y[:N], refY, BF16_ONCE if dtype == "bf16" else F32_TOL)
    if accumulate:
        refG = refG + old
    close(G, refG, BF16_ONCE if grad == "bf16" else F32_TOL, floor=1e-30)
    return rawY, rawG


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,grad", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (1, 65, 32), (16, 3, 7), (17, 300, 64), (255, 65, 33),
                                   (1000, 512, 130), (1024, 511, 520), (8192, 70000, 16),
                                   (8193, 1000, 24), (20000, 300000, 9), (2048, 700, 1040),
                                   (2049, 700, 1040), (9000, 5000, 1029)])
def test_embedding(N, V, D, dtype, grad):
    r = np.random.default_rng(N + V)
    ids = np.minimum((V ** r.random(N)).astype(np.int64) - 1, V - 1)
    run_embedding(ids, V, D, dtype, grad, ldx=0 if N % 2 else 3)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [5, 400, 2100, 9000])
@pytest.mark.parametrize("kind", ["all_same", "padding", "all_padding", "descending", "ends"])
def test_embedding_orders(N, kind):
    V, D = 50, 40
    ids = np.full(N, 7)
    if kind == "padding":
        ids = np.arange(N) % V
        ids[::3], ids[1::7] = -1, V
        ids[-1] = 2 ** 31 - 1
    elif kind == "all_padding":
        ids[:] = -5
    elif kind == "descending":
        ids = (N - 1 - np.arange(N)) * V // N
    elif kind == "ends":
        ids = np.where(np.arange(N) < N // 2, 0, V - 1)
    run_embedding(ids, V, D, "f32", "f32")
    run_embedding(ids, V, D, "bf16", "bf16", accumulate=True)


@pytest.mark.gpu
@pytest.mark.parametrize("grad", ["f32", "bf16"])
@pytest.mark.parametrize("off", [0, 1, 5, 33])
@pytest.mark.parametrize("N,V,D", [(0, 3000, 61), (6, 20000, 61), (6, 9, 1), (40, 70000, 7)])
def test_embedding_clears_a_table_without_gaps(N, V, D, off, grad):
    """Tables that begin at any value: every row is written, and nothing before or behind them."""
    t, fill = (np.uint16, 0x7FC0) if grad == "bf16" else (np.float32, np.float32(7))
    r = np.random.default_rng(N)
    ids, dY = r.integers(0, V, N), r.integers(-8, 9, (max(N, 1), D)).astype(np.float32)   # exact in both
    dYb = store(dY, grad)[0]
    full = DB.from_numpy(np.full(V * D + off + 300, fill, t))
    hip.embedding_bwd(DT[grad], N, V, D, 1.0, ints(ids if N else [0]), dYb, D,
                      full.ptr + off * np.dtype(t).itemsize, D, DT[grad], False, None, 0)
    raw = full.numpy()
    assert (raw[:off] == fill).all() and (raw[off + V * D:] == fill).all()
    got = raw[off:off + V * D].reshape(V, D)
    want = emb_ref(ids, np.zeros((V, D)), dY[:N].astype(np.float64), 1.0)[1]
    assert ((bits_to_f32(got) if grad == "bf16" else got) == want).all()


@pytest.mark.gpu
def test_embedding_no_tokens():
    run_embedding([], 5, 12, "f32", "f32")
    run_embedding([], 5, 12, "bf16", "f32", accumulate=True)


@pytest.mark.gpu
def test_embedding_accumulate_leaves_other_rows():
    """Rows without a token are not touched, NaN in them included; reruns are bit-identical."""
    V, D, N = 40, 20, 300
    ids = np.random.default_rng(3).integers(0, 10, N)
    r = np.random.default_rng(4)
    dYb, dY = store(r.standard_normal((N, D)), "f32")
    old = np.full((V, D), np.nan, np.float32)
    old[:10] = 1.0
    size = hip.embedding_bwd_workspace(N, V, D)
    ws, ib = DB(size), ints(ids)
    raws = []
    for _ in range(3):
        gb = DB.from_numpy(old)
        hip.embedding_bwd(hip.F32, N, V, D, 1.0, ib, dYb, D, gb, D, hip.F32, True, ws, size)
        raws.append(gb.numpy())
    assert np.isnan(raws[0][10:]).all()
    close(raws[0][:10].astype(np.float64), emb_ref(ids, np.zeros((V, D)), dY, 1.0)[1][:10] + 1.0, F32_TOL)
    assert all((x[:10] == raws[0][:10]).all() for x in raws)


# ------------------------------------------------------------------------------ the losses

def loss_ref(H, W, q, c, factor, wscale, dloss, keep):
    """q: N x V target probabilities; rows not in keep are padding."""
    z = c * (H[keep] @ W.T)
    m = z.max(1, keepdims=True)
    lse = (m + np.log(np.exp(z - m).sum(1, keepdims=True)))
    qk = q[keep]
    logq = np.log(np.where(qk > 0, qk, 1.0))
    loss = factor * (qk * (logq - z + lse)).sum(1)
    G = (np.exp(z - lse) - qk) * (dloss[keep, None] * wscale)
    N, D = H.shape
    out = [np.zeros(N), np.zeros(N), np.zeros((N, D))]
    out[0][keep], out[1][keep], out[2][keep] = loss, lse[:, 0], G @ W
    return out + [G.T @ H[keep]]


class Loss:
    """A loss's inputs on the device, and its calls."""

    def __init__(self, N, V, D, dtype, K=None, T=1.0, scale=1.0, pad=0.0, ldx=0, seed=0, hard=4.0):
        r = np.random.default_rng(seed)
        self.N, self.V, self.D, self.dtype, self.K, self.T, self.scale = N, V, D, dtype, K, T, scale
        self.ld = D + ldx
        W = r.standard_normal((V, D)) * 0.1
        target = r.integers(0, V, N)
        # logits of a spread of about 2 around a target between likely and not
        H = r.standard_normal((N, D)) * (20.0 / np.sqrt(D))
        H += W[target] * (r.random((N, 1)) * hard * 100.0 / D)
        pads = r.random(N) < pad
        self.Hb, self.H = store(H, dtype, self.ld)
        self.Wb, self.W = store(W, dtype, self.ld)
        self.dloss = (r.random(N) + 0.5).astype(np.float32)
        self.dlb = DB.from_numpy(self.dloss)
        if K is None:
            target[pads] = np.where(np.arange(N)[pads] % 2 == 0, -1, V + 3)
            self.keep = ~pads
            q = np.zeros((N, V))
            q[np.arange(N)[self.keep], target[self.keep]] = 1.0
            self.ids = ints(target)
        else:
            idx = r.integers(0, V, (N, K))          # some twice in a row
            top = r.standard_normal((N, K)) * 2 + 5
            idx[:, 0] = target
            out = r.random((N, K)) < 0.2
            idx[out] = np.where(r.random((N, K)) < 0.5, -1, V)[out]
            top[r.random((N, K)) < 0.1] = -np.inf
            idx[pads] = -1
            top = top.astype(np.float32)
            ok = (idx >= 0) & (idx < V) & (top > -np.inf)
            self.keep = ok.any(1)
            y = np.where(ok, top.astype(np.float64) / T, -np.inf)
            y[~self.keep] = 0.0
            e = np.where(ok, np.exp(y - y.max(1, keepdims=True)), 0.0)
            e /= np.maximum(e.sum(1, keepdims=True), 1e-300)
            self.qk = e
            q = np.zeros((N, V))
            for k in range(K):
                at = ok[:, k]
                np.add.at(q, (np.arange(N)[at], idx[at, k]), e[at, k])
            self.idx, self.ok = idx, ok
            self.ids, self.top = ints(idx), DB.from_numpy(top)
        self.q = q

    def ref(self):
        if self.K is None:
            return loss_ref(self.H, self.W, self.q, self.scale, 1.0, self.scale, self.dloss, self.keep)
        # a token that occurs twice: its entries' own log q, its summed probability in G
        out = loss_ref(self.H, self.W, self.q, 1 / self.T, self.T ** 2, self.T, self.dloss, self.keep)
        z = self.H @ self.W.T / self.T
        for n in np.nonzero(self.keep)[0]:
            k = self.ok[n]
            qk, zk = self.qk[n][k], z[n][self.idx[n][k]]
            logq = np.log(np.where(qk > 0, qk, 1.0))
            out[0][n] = self.T ** 2 * (qk * (logq - zk + out[1][n])).sum()
        return out

    def head(self):
        if self.K is None:
            return (DT[self.dtype], self.N, self.V, self.D, self.scale, self.Hb, self.ld, self.Wb, self.ld,
                    self.ids)
        return (DT[self.dtype], self.N, self.V, self.D, self.K, self.T, self.Hb, self.ld, self.Wb, self.ld,
                self.ids, self.top)

    def least(self, backward):
        if self.K is None:
            return hip.linear_xent_workspace(DT[self.dtype], self.N, self.V, self.D, backward)
        return hip.linear_distill_workspace(DT[self.dtype], self.N, self.V, self.D, self.K, backward)

    def fwd(self, loss, lse, ws, size):
        (hip.linear_xent_fwd if self.K is None else hip.linear_distill_fwd)(*self.head(), loss, lse, ws,
                                                                           size)

    def bwd(self, lse, dloss, dH, lddh, acc_dH, dW, lddw, acc_dW, gtype, ws, size):
        (hip.linear_xent_bwd if self.K is None else hip.linear_distill_bwd)(
            *self.head(), lse, dloss, dH, lddh, acc_dH, dW, lddw, acc_dW, gtype, ws, size)


def run_loss(c, grad=None, extra=0, accumulate=False):
    """Forward and backward in `extra` bytes above the least workspace; compares all four results."""
    grad = grad or c.dtype
    N, V, D, ld = c.N, c.V, c.D, c.ld
    loss, lse = (DB.from_numpy(np.full(N, np.nan, np.float32)) for _ in range(2))
    size = max(c.least(0), c.least(1)) + extra
    ws = DB(size)
    r = np.random.default_rng(9)
    old = [r.standard_normal(s) * 0.1 if accumulate else np.full(s, np.nan) for s in ((N, D), (V, D))]
    bufs = [store(x, grad, ld) for x in old]
    c.fwd(loss, lse, ws, size)
    c.bwd(lse, c.dlb, bufs[0][0], ld, accumulate, bufs[1][0], ld, accumulate, DT[grad], ws, size)
    ref = c.ref()
    got = [loss.numpy().astype(np.float64), lse.numpy().astype(np.float64)]
    for (b, _), shape in zip(bufs, ((N, D), (V, D))):
        x, raw = fetch(b, shape, grad, ld)
        gap = raw[:, D:]
        assert (gap == 0x7FC0).all() if grad == "bf16" else np.isnan(gap).all()
        got.append(x)
    close(got[0], ref[0], F32_TOL, floor=1.0)
    close(got[1], ref[1], F32_TOL, floor=1.0)
    for k in (0, 1):
        want = ref[2 + k] + (bufs[k][1] if accumulate else 0.0)
        tol = F32_TOL if c.dtype == "f32" else BF16_TOL
        # p and q are good to that much of 1, so a gradient is of the largest weight times operand
        weight = c.dloss.max() * (c.scale if c.K is None else c.T)
        close(got[2 + k], want, tol, floor=weight * np.abs((c.W, c.H)[k]).max())
    assert (got[0][~c.keep] == 0).all() and (got[1][~c.keep] == 0).all()
    if not accumulate:
        assert (got[2][~c.keep] == 0).all()
    return got


SHAPES = [(1, 1, 1), (1, 65, 32), (2, 3, 5), (31, 257, 64), (64, 1000, 100), (256, 256, 32),
          (257, 300, 40), (300, 1025, 96), (513, 130, 264), (3, 5000, 72), (16, 3000, 129),
          (5, 64, 1030), (9, 700, 300), (17, 3000, 129), (5, 70000, 61), (16, 65600, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("N,V,D", SHAPES)
def test_xent(N, V, D, dtype):
    run_loss(Loss(N, V, D, dtype, scale=1.0 if N % 2 else 0.5, pad=0.25 if N > 2 else 0.0,
                  ldx=0 if V % 2 else 5))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("N,V,D", SHAPES)
@pytest.mark.parametrize("K,T", [(1, 1.0), (7, 2.0), (130, 0.5)])
def test_distill(N, V, D, K, T, dtype):
    if K > 7 and N * V > 100000:
        K = 70
    run_loss(Loss(N, V, D, dtype, K=K, T=T, pad=0.25 if N > 2 else 0.0, ldx=0 if V % 2 else 8))


@pytest.mark.gpu
@pytest.mark.parametrize("K", [None, 5])
@pytest.mark.parametrize("dtype,grad", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("extra", [0, 1 << 20, 64 << 20])
def test_loss_pieces_and_accumulation(K, dtype, grad, extra):
    """The vocabulary in pieces of one block of rows up to all of it gives the same; gradients add."""
    c = Loss(300, 2900, 72, dtype, K=K, T=1.5, pad=0.3, ldx=8)
    run_loss(c, grad, extra)
    run_loss(c, grad, extra, accumulate=True)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [None, 4])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_loss_padding_holds_anything(K, dtype):
    """NaN and infinities in padded rows of H and of dloss reach nothing; all rows padded is fine."""
    c = Loss(200, 300, 48, dtype, K=K, pad=0.5)
    clean = run_loss(c)
    H = c.H.copy()
    H[~c.keep] = np.where(np.arange((~c.keep).sum())[:, None] % 2 == 0, np.nan, np.inf)
    c.Hb, _ = store(H, dtype)
    d = c.dloss.copy()
    d[~c.keep] = np.nan
    c.dlb = DB.from_numpy(d)
    for a, b in zip(clean, run_loss(c)):
        assert (a == b).all()
    c.ids = ints(np.full(c.N * (K or 1), -1))
    c.keep[:] = False
    c.q[:] = 0
    if K:
        c.ok[:] = False
    c.H = np.zeros_like(c.H)
    run_loss(c)


@pytest.mark.gpu
def test_xent_extremes():
    """Huge and tiny logits: a sure target, a hopeless one, fp32 values near the type's ends."""
    N, V, D = 40, 600, 16
    c = Loss(N, V, D, "f32", seed=5)
    H = c.H.copy()
    H[:10] *= 50.0
    H[10:20] *= 1e-30
    c.Hb, c.H = store(H, "f32")
    # a logit of 1000 is good to sqrt(D) u of 1000, and its probability to as much absolute
    loss, lse = DB.empty((N,), np.float32), DB.empty((N,), np.float32)
    size = c.least(1) + (1 << 20)
    ws = DB(size)
    dH, dW = DB.empty((N, D), np.float32), DB.empty((V, D), np.float32)
    c.fwd(loss, lse, ws, size)
    c.bwd(lse, c.dlb, dH, D, False, dW, D, False, hip.F32, ws, size)
    ref = c.ref()
    zmax = np.abs(c.H @ c.W.T).max()
    tol = 4 * 4 * zmax * 2.0 ** -24
    assert zmax > 200
    close(loss.numpy().astype(np.float64), ref[0], tol / max(1.0, np.abs(ref[0]).max()), floor=1.0)
    close(dH.numpy().astype(np.float64), ref[2], 2 * tol)
    close(dW.numpy().astype(np.float64), ref[3], 2 * tol)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [-100, -30, 60, 100])
def test_loss_operands_of_any_scale(k):
    """H 2^k and W 2^-k have the logits, the losses and, scaled back, the gradients of H and W, bit
    for bit: the products take each row at a scale of its own."""
    outs = []
    for j in (0, k):
        c = Loss(70, 300, 40, "f32", seed=3)
        H, W = np.ldexp(c.H, j), np.ldexp(c.W, -j)
        c.Hb, c.H = store(H, "f32")
        c.Wb, c.W = store(W, "f32")
        size = max(c.least(0), c.least(1))
        ws = DB(size)
        loss, lse = DB.empty((c.N,), np.float32), DB.empty((c.N,), np.float32)
        dH, dW = DB.empty((c.N, c.D), np.float32), DB.empty((c.V, c.D), np.float32)
        c.fwd(loss, lse, ws, size)
        c.bwd(lse, c.dlb, dH, c.D, False, dW, c.D, False, hip.F32, ws, size)
        outs.append([loss.numpy(), lse.numpy(), np.ldexp(dH.numpy(), j), np.ldexp(dW.numpy(), -j)])
    for a, b in zip(*outs):
        assert (a == b).all()


@pytest.mark.gpu
def test_loss_rows_of_many_scales():
    """Rows of H and of W, and loss weights, whose sizes differ by factors of up to 2^24."""
    N, V, D = 150, 400, 48
    c = Loss(N, V, D, "f32", seed=4)
    r = np.random.default_rng(5)
    c.Hb, c.H = store(np.ldexp(c.H, -r.integers(0, 24, (N, 1))), "f32")
    c.Wb, c.W = store(np.ldexp(c.W, -r.integers(0, 24, (V, 1))), "f32")
    c.dloss = np.ldexp(c.dloss, -r.integers(0, 24, N)).astype(np.float32)
    c.dlb = DB.from_numpy(c.dloss)
    got = run_loss(c)
    ref = c.ref()
    # every row of dH to its own size, as its sum's terms have the row's weight
    err = np.abs(got[2] - ref[2]).max(1) / (c.dloss * np.abs(c.W).max())
    assert err.max() <= F32_TOL, err.max()


@pytest.mark.gpu
@pytest.mark.parametrize("K", [None, 6])
def test_loss_gradient_against_differences(K):
    """dH and dW against central differences of the forward's own losses, step 2^-5: the second
    difference leaves step^2 / 6 of the third derivative, and fp32 losses of about 5 a noise of
    5 * 2^-23 / step per row."""
    N, V, D = 6, 50, 8
    c = Loss(N, V, D, "f32", K=K, T=1.3, seed=2)
    size = max(c.least(0), c.least(1))
    ws = DB(size)
    loss, lse = DB.empty((N,), np.float32), DB.empty((N,), np.float32)
    dH, dW = DB.empty((N, D), np.float32), DB.empty((V, D), np.float32)
    c.fwd(loss, lse, ws, size)
    c.bwd(lse, None, dH, D, False, dW, D, False, hip.F32, ws, size)
    gH, gW = dH.numpy(), dW.numpy()
    H0, W0 = c.H.astype(np.float32), c.W.astype(np.float32)
    step = np.float32(2.0 ** -5)

    def total(H, W):
        c.Hb, c.Wb = DB.from_numpy(H), DB.from_numpy(W)
        c.fwd(loss, None, ws, size)
        return loss.numpy().astype(np.float64).sum()

    for n, d in ((0, 0), (3, 5), (5, 7)):
        a, b = H0.copy(), H0.copy()
        a[n, d] += step
        b[n, d] -= step
        diff = (total(a, W0) - total(b, W0)) / (float(a[n, d]) - float(b[n, d]))
        assert abs(diff - gH[n, d]) <= 2e-3 * max(1.0, np.abs(gH).max())
    for v, d in ((0, 0), (int(np.argmax(np.abs(gW).max(1))), 3), (V - 1, 7)):
        a, b = W0.copy(), W0.copy()
        small = np.float32(2.0 ** -8)     # H is about 7: the same change of a logit
        a[v, d] += small
        b[v, d] -= small
        diff = (total(H0, a) - total(H0, b)) / (float(a[v, d]) - float(b[v, d]))
        assert abs(diff - gW[v, d]) <= 4e-3 * max(1.0, np.abs(gW).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("N", [1, 4, 8, 16, 18, 32, 33])
@pytest.mark.parametrize("D", [40, 77])
def test_few_rows_of_a_long_table(N, D, dtype):
    """V above 2^14, where few rows take the table in blocks of 64 of its rows; D = 77 takes 16-bit
    tables at odd addresses."""
    run_loss(Loss(N, 17001, D, dtype, pad=0.2 if N > 2 else 0.0))
    run_loss(Loss(N, 17001, D, dtype, K=9, T=2.0, pad=0.2 if N > 2 else 0.0), accumulate=True)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [None, 4])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("N", [5, 13, 29])
def test_few_rows_padding_holds_anything(N, K, dtype):
    c = Loss(N, 300, 47, dtype, K=K, pad=0.5, seed=1)
    assert c.keep.any() and not c.keep.all()
    clean = run_loss(c)
    H = c.H.copy()
    H[~c.keep] = np.where(np.arange((~c.keep).sum())[:, None] % 2 == 0, np.nan, np.inf)
    c.Hb, _ = store(H, dtype)
    d = c.dloss.copy()
    d[~c.keep] = np.nan
    c.dlb = DB.from_numpy(d)
    for a, b in zip(clean, run_loss(c)):
        assert (a == b).all()
    c.ids = ints(np.full(c.N * (K or 1), -1))
    c.keep[:] = False
    c.q[:] = 0
    if K:
        c.ok[:] = False
    c.H = np.zeros_like(c.H)
    run_loss(c)


@pytest.mark.gpu
def test_few_rows_of_a_table_past_the_short_form():
    """V above 2^21: the form for many rows also takes few of them."""
    run_loss(Loss(2, (1 << 21) + 3, 8, "bf16"), "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("K", [None, 3])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("N,V,D", [(7, 500, 40), (130, 700, 96), (300, 5000, 200)])
def test_loss_without_some_results(N, V, D, K, dtype):
    """lse, dH, dW and dloss may be missing: what is left does not change, nor does a second run."""
    c = Loss(N, V, D, dtype, K=K, pad=0.2)
    size = max(c.least(0), c.least(1)) + (4 << 20)
    ws = DB(size)
    t = np.uint16 if dtype == "bf16" else np.float32

    def run(with_lse, with_H, with_W, dloss):
        loss, lse = (DB.from_numpy(np.zeros(N, np.float32)) for _ in range(2))
        dH, dW = DB.from_numpy(np.zeros((N, D), t)), DB.from_numpy(np.zeros((V, D), t))
        c.fwd(loss, lse if with_lse else None, ws, size)
        if not with_lse:
            return loss.numpy(), None, None
        c.bwd(lse, dloss, dH if with_H else None, D, False, dW if with_W else None, D, False, DT[dtype],
              ws, size)
        return loss.numpy(), dH.numpy(), dW.numpy()

    both = run(True, True, True, c.dlb)
    assert all((a == b).all() for a, b in zip(both, run(True, True, True, c.dlb)))
    assert (run(False, True, True, c.dlb)[0] == both[0]).all()
    assert (run(True, True, False, c.dlb)[1] == both[1]).all()
    assert (run(True, False, True, c.dlb)[2] == both[2]).all()
    run(True, False, False, c.dlb)
    ones = run(True, True, True, DB.from_numpy(np.ones(N, np.float32)))
    assert all((a == b).all() for a, b in zip(ones, run(True, True, True, None)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,grad", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("weights", ["equal", "zero", "tiny", "wide"])
def test_loss_weights(weights, dtype, grad):
    """One loss weight for all rows as a mean has it, none, tiny ones, and weights of both signs over
    a range of 2^40: the gradients hold what they hold for weights of about 1."""
    N, V, D = 150, 400, 48
    c = Loss(N, V, D, dtype, seed=6, pad=0.1)
    r = np.random.default_rng(7)
    c.dloss = {"equal": np.full(N, 1 / 1719), "zero": np.zeros(N), "tiny": np.full(N, 2.0 ** -100) * (1 + r.random(N)),
               "wide": np.ldexp(r.standard_normal(N), r.integers(-40, 1, N))}[weights].astype(np.float32)
    c.dlb = DB.from_numpy(c.dloss)
    size = max(c.least(0), c.least(1))
    ws = DB(size)
    loss, lse = DB.empty((N,), np.float32), DB.empty((N,), np.float32)
    bufs = [store(np.full(s, np.nan), grad)[0] for s in ((N, D), (V, D))]
    c.fwd(loss, lse, ws, size)
    c.bwd(lse, c.dlb, bufs[0], D, False, bufs[1], D, False, DT[grad], ws, size)
    ref, tol = c.ref(), F32_TOL if dtype == "f32" else BF16_TOL
    for k in (0, 1):
        got = fetch(bufs[k], ((N, D), (V, D))[k], grad)[0]
        close(got, ref[2 + k], tol, floor=np.abs(c.dloss).max() * np.abs((c.W, c.H)[k]).max())
        if weights == "zero":
            assert (got == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("K", [None, 3])
@pytest.mark.parametrize("dtype,grad", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16")])
def test_loss_of_no_rows(K, dtype, grad):
    """Nothing is read; dW is zero, or stays as it was where it is added to."""
    V, D, ld = 70, 33, 35
    t = np.uint16 if grad == "bf16" else np.float32
    for acc in (False, True):
        dW = DB.from_numpy(np.full((V, ld), 7, t))
        head = (DT[dtype], 0, V, D) + ((1.0,) if K is None else (K, 2.0)) + (None, D, None, D)
        ids = (None,) if K is None else (None, None)
        if K is None:
            hip.linear_xent_fwd(*head, *ids, None, None, None, 0)
            hip.linear_xent_bwd(*head, *ids, None, None, None, D, False, dW, ld, acc, DT[grad], None, 0)
        else:
            hip.linear_distill_fwd(*head, *ids, None, None, None, 0)
            hip.linear_distill_bwd(*head, *ids, None, None, None, D, False, dW, ld, acc, DT[grad], None, 0)
        got = dW.numpy()
        assert (got[:, :D] == (7 if acc else 0)).all() and (got[:, D:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("N,V,D,ldx", [(1, 300, 40, 0), (7, 17001, 24, 3), (16, 129, 700, 0)])
def test_few_rows_with_gradients_in_floats(N, V, D, ldx, accumulate):
    run_loss(Loss(N, V, D, "bf16", ldx=ldx), "f32", accumulate=accumulate)
    run_loss(Loss(N, V, D, "bf16", K=5, T=2.0, ldx=ldx), "f32", accumulate=accumulate)


def part(buf, first, rows, D, dtype):
    """Rows first .. first + rows - 1 of a large device matrix of rows of D values."""
    t = np.dtype(np.uint16 if dtype == "bf16" else np.float32)
    out = np.empty((rows, D), t)
    hip.check(hip.load().dh_memcpy_d2h(out.ctypes.data, buf.ptr + first * D * t.itemsize, out.nbytes), "d2h")
    return (bits_to_f32(out) if dtype == "bf16" else out).astype(np.float64)


@pytest.mark.gpu
def test_table_past_32_bit_offsets():
    """V D above 2^31: rows at the table's ends.  The table repeats with a period, so the reference
    needs one period and how often each of its rows occurs."""
    V, D, P = 262200, 8200, 97
    assert V * D > 2 ** 31
    r = np.random.default_rng(1)
    pat = bf16_bits((r.standard_normal((P, D)) * 0.1).astype(np.float32))
    Wp = bits_to_f32(pat).astype(np.float64)
    W = np.empty((V, D), np.uint16)
    for s in range(0, V, P):
        W[s:s + P] = pat[:V - s]
    Wb = DB.from_numpy(W)
    del W
    times = np.bincount(np.arange(V) % P, minlength=P)
    dWb = DB(V * D * 2)
    edge = 300
    spots = np.concatenate([np.arange(edge), np.arange(V - edge, V)])
    for N in (3, 20):
        Hb, H = store(r.standard_normal((N, D)) * (20.0 / np.sqrt(D)), "bf16")
        target = spots[r.integers(0, 2 * edge, N)]
        target[:3] = V - 1, 0, V - 2
        size = max(hip.linear_xent_workspace(hip.BF16, N, V, D, b) for b in (0, 1)) + (64 << 20)
        ws, tb = DB(size), ints(target)
        loss, lse = DB.empty((N,), np.float32), DB.empty((N,), np.float32)
        dHb = store(np.zeros((N, D)), "bf16")[0]
        hip.linear_xent_fwd(hip.BF16, N, V, D, 1.0, Hb, D, Wb, D, tb, loss, lse, ws, size)
        hip.linear_xent_bwd(hip.BF16, N, V, D, 1.0, Hb, D, Wb, D, tb, lse, None, dHb, D, False, dWb, D, False,
                            hip.BF16, ws, size)
        z = H @ Wp.T
        m = z.max(1, keepdims=True)
        rl = (m + np.log((times * np.exp(z - m)).sum(1, keepdims=True)))
        p = np.exp(z - rl)
        close(lse.numpy().astype(np.float64), rl[:, 0], F32_TOL)
        close(loss.numpy().astype(np.float64), rl[:, 0] - z[np.arange(N), target % P], F32_TOL)
        G = np.zeros((N, 2 * edge))
        G[:] = p[:, spots % P]
        for n in range(N):
            G[n, np.searchsorted(spots, target[n])] -= 1.0
        close(fetch(dHb, (N, D), "bf16")[0], (p * times) @ Wp - Wp[target % P], BF16_TOL, floor=np.abs(Wp).max())
        got = np.concatenate([part(dWb, 0, edge, D, "bf16"), part(dWb, V - edge, edge, D, "bf16")])
        close(got, G.T @ H, BF16_TOL, floor=np.abs(H).max())
        # the embedding of the same tokens, and its gradient over what is there
        Yb = store(np.zeros((N, D)), "bf16")[0]
        hip.embedding_fwd(hip.BF16, N, V, D, 2.0, tb, Wb, D, Yb, D)
        close(fetch(Yb, (N, D), "bf16")[0], 2.0 * Wp[target % P], BF16_ONCE)
        hip.embedding_bwd(hip.BF16, N, V, D, 1.0, tb, Hb, D, dWb, D, hip.BF16, False, ws, size)
        want = np.zeros((2 * edge, D))
        np.add.at(want, np.searchsorted(spots, target), H)
        got = np.concatenate([part(dWb, 0, edge, D, "bf16"), part(dWb, V - edge, edge, D, "bf16")])
        close(got, want, BF16_ONCE)


# ------------------------------------------------------------------------------ together

class Tied:
    """A small language model's two ends, fp32: x = s W[id], y = its layer norm, h = y P, cross entropy
    and distillation of h W^T, and the gradients of W (from all three) and of P."""
    N, V, D, K, S, T = 96, 500, 64, 4, 8.0, 2.0

    def __init__(self):
        r = np.random.default_rng(11)
        N, V, D, K = self.N, self.V, self.D, self.K
        self.W0 = (r.standard_normal((V, D)) * 0.2).astype(np.float32)
        self.P0 = (r.standard_normal((D, D)) * 0.2).astype(np.float32)
        self.id0 = r.integers(0, V, N)
        self.t0 = r.integers(0, V, N)
        self.id0[-5:] = self.t0[-5:] = -1           # the batch's padding
        self.top0 = np.argsort(r.random((N, V)), 1)[:, :K]
        self.top0[-5:] = -1
        self.logit0 = (r.standard_normal((N, K)) * 2).astype(np.float32)
        self.w1, self.w2 = np.full(N, 0.7 / N, np.float32), np.full(N, 0.3 / N, np.float32)
        up = DB.from_numpy
        self.W, self.P, self.id, self.t = up(self.W0), up(self.P0), ints(self.id0), ints(self.t0)
        self.top, self.logit, self.a, self.b = ints(self.top0), up(self.logit0), up(self.w1), up(self.w2)
        f = lambda *s: DB.empty(s, np.float32)  # noqa: E731
        self.x, self.y, self.h, self.dh, self.dy, self.dx = (f(N, D) for _ in range(6))
        self.dW, self.dP = f(V, D), f(D, D)
        self.l1, self.l2, self.lse1, self.lse2 = (f(N) for _ in range(4))
        self.size = max(hip.embedding_bwd_workspace(N, V, D),
                        *(hip.linear_xent_workspace(0, N, V, D, b) for b in (0, 1)),
                        *(hip.linear_distill_workspace(0, N, V, D, K, b) for b in (0, 1)))
        self.ws = DB(self.size)

    def head(self, backward):
        N, V, D, F = self.N, self.V, self.D, hip.F32
        w = (self.ws, self.size)
        x = (F, N, V, D, 1.0, self.h, D, self.W, D, self.t)
        d = (F, N, V, D, self.K, self.T, self.h, D, self.W, D, self.top, self.logit)
        hip.linear_xent_fwd(*x, self.l1, self.lse1, *w)
        hip.linear_distill_fwd(*d, self.l2, self.lse2, *w)
        if backward:
            hip.linear_xent_bwd(*x, self.lse1, self.a, self.dh, D, False, self.dW, D, False, F, *w)
            hip.linear_distill_bwd(*d, self.lse2, self.b, self.dh, D, True, self.dW, D, True, F, *w)

    def step(self):
        N, V, D, F = self.N, self.V, self.D, hip.F32
        hip.embedding_fwd(F, N, V, D, self.S, self.id, self.W, D, self.x, D)
        hip.layer_norm(self.x, self.y, N, D)
        hip.gemm_f32(False, False, N, D, D, self.y, D, self.P, D, 0.0, self.h, D)
        self.head(True)
        hip.gemm_f32(True, False, D, D, N, self.y, D, self.dh, D, 0.0, self.dP, D)
        hip.gemm_f32(False, True, N, D, D, self.dh, D, self.P, D, 0.0, self.dy, D)
        hip.layer_norm_bwd(self.x, self.y, self.dy, self.dx, N, D)
        hip.embedding_bwd(F, N, V, D, self.S, self.id, self.dx, D, self.dW, D, F, True, self.ws, self.size)

    def ref(self):
        N, V, D = self.N, self.V, self.D
        W, P = self.W0.astype(np.float64), self.P0.astype(np.float64)
        x, _ = emb_ref(self.id0, W, np.zeros((N, D)), self.S)
        inv = 1 / np.sqrt(x.var(1, keepdims=True) + 1e-5)
        y = (x - x.mean(1, keepdims=True)) * inv
        h, keep = y @ P, self.t0 >= 0
        q1, q2 = np.zeros((N, V)), np.zeros((N, V))
        q1[np.nonzero(keep)[0], self.t0[keep]] = 1
        e = np.exp(self.logit0.astype(np.float64) / self.T)
        np.put_along_axis(q2, np.maximum(self.top0, 0), e / e.sum(1, keepdims=True), 1)
        r1 = loss_ref(h, W, q1, 1.0, 1.0, 1.0, self.w1, keep)
        r2 = loss_ref(h, W, q2, 1 / self.T, self.T ** 2, self.T, self.w2, keep)
        dh = r1[2] + r2[2]
        dy = dh @ P.T
        dx = inv * (dy - dy.mean(1, keepdims=True) - y * (dy * y).mean(1, keepdims=True))
        return r1[0], r2[0], r1[3] + r2[3] + emb_ref(self.id0, W, dx, self.S)[1], y.T @ dh


@pytest.mark.gpu
def test_tied_table_step():
    """Four kinds of step between the losses and the result, each good to F32_TOL of its largest
    value, which is up to four times a typical one: 16 F32_TOL of the results' largest."""
    m = Tied()
    m.step()
    got = [b.numpy().astype(np.float64) for b in (m.l1, m.l2, m.dW, m.dP)]
    for g, want in zip(got, m.ref()):
        close(g, want, 16 * F32_TOL)
    # steps against the gradient lower the loss: the directional derivative over a small step of W
    # as the embedding and both heads see it, second order below 1e-2 of it
    total = lambda: float(m.w1 @ m.l1.numpy().astype(np.float64) + m.w2 @ m.l2.numpy().astype(np.float64))  # noqa: E731
    before, g = total(), got[2]
    step = 1e-2 / np.linalg.norm(g)
    moved = []
    for s in (1, -1):
        m.W = DB.from_numpy((m.W0 + s * step * g).astype(np.float32))
        m.step()
        moved.append(total())
    slope = (moved[0] - moved[1]) / (2 * step)
    assert moved[1] < before < moved[0]
    assert abs(slope - (g * g).sum()) <= 1e-2 * (g * g).sum()


def _runtime():
    rt = ctypes.CDLL("libamdhip64.so")
    v, p = ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p)
    for name, args in (("hipStreamCreate", [p]), ("hipStreamDestroy", [v]), ("hipStreamSynchronize", [v]),
                       ("hipStreamBeginCapture", [v, ctypes.c_int]), ("hipStreamEndCapture", [v, p]),
                       ("hipGraphInstantiate", [p, v, v, v, ctypes.c_size_t]), ("hipGraphLaunch", [v, v]),
                       ("hipGraphExecDestroy", [v]), ("hipGraphDestroy", [v])):
        f = getattr(rt, name)
        f.restype, f.argtypes = ctypes.c_int, args
    return rt


class Recorded:
    """A loss's forward and backward and an embedding's, with a workspace of their own."""

    def __init__(self, N, V, D, dtype, K, seed):
        self.c = c = Loss(N, V, D, dtype, K=K, pad=0.2, seed=seed)
        t = np.uint16 if dtype == "bf16" else np.float32
        self.size = max(c.least(0), c.least(1), hip.embedding_bwd_workspace(N, V, D)) + (1 << 20)
        self.ws = DB(self.size)
        self.id = ints(np.random.default_rng(seed).integers(-1, V, N))
        self.out = [DB.empty((N,), np.float32), DB.empty((N,), np.float32), DB.empty((N, D), t), DB.empty((V, D), t),
                    DB.empty((N, D), t), DB.empty((V, D), t)]

    def run(self):
        c, (loss, lse, dH, dW, Y, dE) = self.c, self.out
        dt = DT[c.dtype]
        c.fwd(loss, lse, self.ws, self.size)
        c.bwd(lse, c.dlb, dH, c.D, False, dW, c.D, False, dt, self.ws, self.size)
        hip.embedding_fwd(dt, c.N, c.V, c.D, 1.0, self.id, c.Wb, c.ld, Y, c.D)
        hip.embedding_bwd(dt, c.N, c.V, c.D, 1.0, self.id, dH, c.D, dE, c.D, dt, False, self.ws, self.size)

    def wipe(self):
        for b in self.out:
            g = np.full(b.shape, 7, b.dtype)
            hip.check(hip.load().dh_memcpy_h2d(b.ptr, g.ctypes.data, g.nbytes), "h2d")
        hip.sync()

    def values(self):
        return [b.numpy() for b in self.out]


@pytest.mark.gpu
@pytest.mark.parametrize("a,b", [((200, 3000, 72, "bf16", None), (12, 900, 50, "f32", 5)),
                                 ((9, 20000, 64, "bf16", 4), (2100, 300, 40, "f32", None)),
                                 ((9000, 40, 24, "bf16", None), (300, 700, 130, "f32", 40))])
def test_graphs_on_other_streams(a, b):
    """Recorded with nothing allocated, on streams of the caller's; two graphs replayed at once, three
    times, their results wiped between: what the library's own stream gives, bit for bit."""
    jobs = [Recorded(*a, seed=1), Recorded(*b, seed=2)]
    want = []
    for j in jobs:
        j.run()
        want.append(j.values())
    R, lib = _runtime(), hip.load()
    streams, graphs, exes = ([ctypes.c_void_p() for _ in jobs] for _ in range(3))
    ref = ctypes.byref
    try:
        for j, s, g, x in zip(jobs, streams, graphs, exes):
            assert R.hipStreamCreate(ref(s)) == 0
            hip.check(lib.dh_set_stream(s), "dh_set_stream")
            j.wipe()
            j.run()                                              # eager on that stream
            assert all(np.array_equal(v, w) for v, w in zip(j.values(), want[jobs.index(j)]))
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
            jobs[0].run()                                        # the program's own work between
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
