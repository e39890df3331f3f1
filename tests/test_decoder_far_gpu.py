"""Rows of the operators around a decoder's attention that lie more than 2^31 values and 2^32 bytes apart."""
import gc

import numpy as np
import pytest

from _decoder import TYPE, U, UB, Cache, attention, floats, ints, norm_rope, quantised, rope_table, rounded, within
from _gpu import DB, bits_to_f32
from dreamcompiler_amd import hip

APART = 2 ** 31 + 64    # values between two rows


@pytest.fixture(autouse=True)
def give_back():
    """The buffers, up to 40 GB, do not wait in the pool for one of the same size."""
    yield
    gc.collect()
    hip.check(hip.load().dh_pool_release(), "dh_pool_release")


class Far:
    """Rows of D values, row i at offsets[i] values of a buffer that nothing else fills."""

    def __init__(self, offsets, x, dtype):
        self.offsets, self.dtype = offsets, dtype
        raw, self.value = rounded(x, dtype)
        self.item, self.D, self.type = raw.itemsize, raw.shape[-1], raw.dtype
        self.buf = DB((max(offsets) + self.D) * self.item)
        for at, row in zip(offsets, raw.reshape(-1, self.D)):
            hip.check(hip.load().dh_memcpy_h2d(self.buf.ptr + at * self.item, np.ascontiguousarray(row).ctypes.data, row.nbytes),
                      "dh_memcpy_h2d")
        hip.sync()

    def get(self):
        out = np.empty((len(self.offsets), self.D), self.type)
        for at, row in zip(self.offsets, out):
            hip.check(hip.load().dh_memcpy_d2h(row.ctypes.data, self.buf.ptr + at * self.item, row.nbytes), "dh_memcpy_d2h")
        return (out if self.item == 4 else bits_to_f32(out)).astype(np.float64).reshape(self.value.shape)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 50])
def test_norm(D):
    """Tokens and sequences far apart, in every tensor."""
    r = np.random.default_rng(0)
    B, S, H, R = 1, 3, 2, 10
    st = (3 * APART, APART, D)
    at = [t * APART + h * D for t in range(S) for h in range(H)]
    x, dy = (r.standard_normal((B, S, H, D)) for _ in range(2))
    X, dY, out, dX = (Far(at, y, "bf16") for y in (x, dy, 0 * x, 0 * x))
    table, pos = rope_table(S, R), np.arange(S)[None]
    a = (hip.BF16, B, S, H, 0, D, R, False, 1e-6, None, floats(table), S, X.buf, st, None, None, None, None)
    hip.qk_norm_rope_fwd(*a, out.buf, st, None, None)
    size = hip.qk_norm_rope_bwd_workspace(D)
    hip.qk_norm_rope_bwd(*a, hip.BF16, dY.buf, st, None, None, hip.BF16, dX.buf, st, None, None, None, None, False, DB(size), size)
    ref = norm_rope(X.value, 1.0, pos, table, R, False, 1e-6)
    within(out.get(), ref, 48 * U * np.abs(ref).max(-1, keepdims=True) * 2 ** 0.5 + UB * np.abs(ref) * (1 + UB))
    dx, _, by, _ = norm_rope(X.value, 1.0, pos, table, R, False, 1e-6, dY.value)
    within(dX.get(), dx, 64 * U * by + UB * (np.abs(dx) + 64 * U * by))


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [0, 1])
def test_cache_and_attention(shift):
    """New tokens, queries and results far apart: rows of whole pieces, and of none."""
    r = np.random.default_rng(1)
    T, Hk, Hq, D, apart = 3, 1, 2, 64, APART + shift
    c = Cache("f8", [T], Hk, D, 16).upload()
    at = [t * apart for t in range(T)]
    K, V = (Far(at, r.standard_normal((T, Hk, D)), "bf16") for _ in "KV")
    st, first = (apart, D), ints([0, T])
    hip.kv_cache_write(hip.BF16, hip.F8, 1, T, Hk, D, K.buf, st, V.buf, st, first, c.lbuf, *c.args())
    held = []
    for x in (K, V):
        codes, s = quantised(x.value, "f8")
        held.append(codes * s.astype(np.float64)[..., None])
    back = [Far(at, np.zeros((T, Hk, D)), "bf16") for _ in "KV"]
    hip.kv_cache_read(hip.BF16, hip.F8, 1, T, Hk, D, back[0].buf, st, back[1].buf, st, first, c.lbuf, *c.args())
    for b, h in zip(back, held):
        assert np.array_equal(b.get(), rounded(h.astype(np.float32), "bf16")[1])
    at = [h * apart for h in range(Hq)]
    Q, O = (Far(at, y, "bf16") for y in (r.standard_normal((1, Hq, D)), np.zeros((1, Hq, D))))
    st = (Hq * apart, apart)
    hip.paged_attention(TYPE["bf16"], hip.F8, 1, Hq, Hk, D, D ** -0.5, 0, Q.buf, st, c.lbuf, 16, *c.args(), O.buf, st, None, None, 0)
    o, _, A = attention(Q.value[0], *held, D ** -0.5)
    dz = (2 * D ** 0.5 + 8) * U * A
    tol = ((2 * dz + 64 * U + 2.0 ** -16) * np.abs(held[1]).max())[:, None]
    within(O.get()[0], o, tol + UB * (np.abs(o) + tol))
