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
          (5, 64, 1030), (9, 700, 300), (17, 3000, 129)]


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
