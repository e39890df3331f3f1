"""Plain 64-bit forms of the norm and rotation of queries and keys, the paged cache and attention over
it, and device buffers with gaps between their rows, for the tests of those operators."""
import numpy as np

from _gpu import DB, bf16_bits, bits_to_f32
from dreamcompiler_amd import hip

U, UB = 2.0 ** -24, 2.0 ** -8       # the largest relative error of one rounding to fp32, to bf16
TYPE = {"f32": hip.F32, "bf16": hip.BF16, "i8": hip.I8, "f8": hip.F8}
TOP = {"i8": 127.0, "f8": 448.0}
RAW = {"f32": np.float32, "bf16": np.uint16, "i8": np.int8, "f8": np.uint8}
NAN = {"f32": np.float32(np.nan), "bf16": np.uint16(0x7FC0)}


def rounded(x, dtype):
    """x as `dtype` holds it: (the stored values, their fp64 meaning)."""
    x = np.asarray(x, np.float32)
    if dtype == "f32":
        return x, x.astype(np.float64)
    bits = bf16_bits(x)
    return bits, bits_to_f32(bits).astype(np.float64)


class Strided:
    """An array of rows of D values on the device, its dimensions in the order `order`, `pad` values
    after each row and NaN in every gap.  `strides` are those of the dimensions as given."""

    def __init__(self, x, dtype, order=None, pad=0):
        raw, self.value = rounded(x, dtype)
        n = raw.ndim - 1
        self.order = tuple(order or range(n))
        self.dtype, self.D, self.shape = dtype, raw.shape[-1], raw.shape
        mixed = raw.transpose(self.order + (n,))
        full = np.full(mixed.shape[:-1] + (self.D + pad,), NAN[dtype], RAW[dtype])
        full[..., :self.D] = mixed
        self.full = full
        self.buf = DB.from_numpy(full if full.size else np.zeros(1, RAW[dtype]))
        step = np.array(full.strides[:-1]) // full.itemsize
        self.strides = tuple(int(step[self.order.index(i)]) for i in range(n))

    @property
    def ptr(self):
        return self.buf.ptr

    _as_parameter_ = ptr    # as ctypes takes it

    def raw(self):
        return self.buf.numpy(self.full.shape, RAW[self.dtype])

    def get(self):
        """The values now, as fp64, in the dimensions' own order; the gaps must be as they were."""
        raw = self.raw()
        gap = raw[..., self.D:]
        assert np.array_equal(gap.view(np.uint8), self.full[..., self.D:].copy().view(np.uint8))
        back = raw[..., :self.D].transpose(tuple(self.order.index(i) for i in range(len(self.order)))
                                           + (len(self.order),))
        return (bits_to_f32(back) if self.dtype == "bf16" else back).astype(np.float64)


def ints(x):
    x = np.asarray(x, np.int32)
    return DB.from_numpy(x if x.size else np.zeros(1, np.int32))


def floats(x):
    return DB.from_numpy(np.asarray(x, np.float32))


def within(got, ref, tol):
    """|got - ref| <= tol everywhere (tol may be an array), non-finite values alike."""
    got, ref = np.asarray(got, np.float64), np.asarray(ref, np.float64)
    fine = np.isfinite(ref)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    assert np.array_equal(got[~fine & ~np.isnan(ref)], ref[~fine & ~np.isnan(ref)])
    over = np.abs(got - ref)[fine] - np.broadcast_to(tol, ref.shape)[fine]
    assert over.size == 0 or over.max() <= 0, float(over.max())


# ------------------------------------------------------------------------------ norm and rotation

def rope_table(P, R, base=10000.0):
    a = np.arange(P)[:, None] * base ** (-2.0 * np.arange(R // 2) / max(R, 1))
    return np.concatenate([np.cos(a), np.sin(a)], 1).astype(np.float32)


def turn(y, cos, sin, R, pairs):
    """y (... x D) with its first R values turned; cos, sin: ... x R / 2."""
    y = y.copy()
    i = np.arange(R // 2)
    at, other = (2 * i, 2 * i + 1) if pairs else (i, i + R // 2)
    a, b = y[..., at].copy(), y[..., other].copy()
    y[..., at], y[..., other] = a * cos - b * sin, b * cos + a * sin
    return y


def norm_rope(x, g, pos, table, R, pairs, eps, dout=None):
    """x: B x S x H x D; pos: B x S.  The output, or with dout (dx, dg, bounds of dx's and dg's terms)."""
    P, D = len(table), x.shape[-1]
    ok = (pos >= 0) & (pos < P)
    rows = table.astype(np.float64)[np.where(ok, pos, 0)][:, :, None, :]
    cos, sin = rows[..., :R // 2], rows[..., R // 2:R]
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    keep = ok[:, :, None, None]
    if dout is None:
        y = x * r * g
        return np.where(keep, turn(y, cos, sin, R, pairs), 0.0)
    dy = np.where(keep, turn(dout, cos, -sin, R, pairs), 0.0)
    xr = x * r
    dyg = dy * g
    dx = r * (dyg - xr * (dyg * xr).mean(-1, keepdims=True))
    size = r * (np.abs(dyg).max(-1, keepdims=True)
                + np.abs(xr).max(-1, keepdims=True) * np.abs(dyg * xr).mean(-1, keepdims=True))
    # A turned value is a sum of two products, each rounded relative to itself, that may cancel: in a row of 1023
    # values, a difference of 0.0023 of products that add up to 0.79 was off by 1.4e-8: 0.3 u of the products, 100 u of
    # the difference.  So the bound of a term of dg counts both products: |a| |c| + |b| |s|, the larger of both signs.
    both = np.maximum(turn(np.abs(dout), np.abs(cos), -np.abs(sin), R, pairs),
                      turn(np.abs(dout), np.abs(cos), np.abs(sin), R, pairs))
    terms = np.where(keep, both * np.abs(xr), 0.0).sum((0, 1, 2))
    return np.where(keep, dx, 0.0), (dy * xr).sum((0, 1, 2)), size, terms


# ------------------------------------------------------------------------------ a paged cache

def e4m3_values():
    """The values of the codes 0 .. 126: 1.4.3 without infinities."""
    code = np.arange(127)
    e, m = code >> 3, code & 7
    return np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))


def quantised(x, kind):
    """(codes as fp64 values, fp32 scales) of rows x (... x D), from the definition."""
    bad = ~np.isfinite(x).all(-1)
    a = np.abs(np.where(np.isfinite(x), x, 0.0))
    s = (a.max(-1) / TOP[kind]).astype(np.float32)
    s64 = np.where(s > 0, s, 1.0).astype(np.float64)[..., None]
    y = np.minimum(a / s64, TOP[kind])
    y = np.where((s > 0)[..., None], y, 0.0)
    values = np.arange(128.0) if kind == "i8" else e4m3_values()
    mid = (values[1:] + values[:-1]) / 2
    n = np.searchsorted(mid, y)
    tie = (n < len(mid)) & (y == mid[np.minimum(n, len(mid) - 1)]) & (n % 2 == 1)
    codes = np.where(np.isnan(x), 0.0, np.sign(x)) * values[n + tie]
    codes[bad] = 0.0
    return codes, np.where(bad, np.float32(np.nan), s)


class Cache:
    """A cache and its table on the device.  Every place starts as `fill` ('nan': what no call may use:
    NaN, or a NaN scale), and `put` writes rows from the host."""

    def __init__(self, kind, lens, Hk, D, page, seed=0, spare=3, ld=None):
        r = np.random.default_rng(seed)
        self.kind, self.Hk, self.D, self.page = kind, Hk, D, page
        held = [-(-max(n, 0) // page) for n in lens]
        self.pages, self.ld = sum(held) + spare, ld or max(1, max(held, default=0))
        ids = r.permutation(self.pages)
        self.table = np.full((max(len(lens), 1), self.ld), -1, np.int32)
        at = 0
        for b, n in enumerate(held):
            self.table[b, :n] = ids[at:at + n]
            at += n
        self.lens = np.asarray(lens, np.int64)
        shape = (self.pages, Hk, page, D)
        self.raw, self.scale = {}, {}
        for n in "KV":
            if kind in TOP:
                self.raw[n] = np.full(shape, 0x55, RAW[kind])
                self.scale[n] = np.full(shape[:3], np.nan, np.float32)
            else:
                self.raw[n] = np.full(shape, NAN[kind], RAW[kind])
        self.bufs = {}

    def put(self, side, b, x, codes_scale=None):
        """Rows x (T x Hk x D) as sequence b's tokens 0 .. T - 1; returns what they stand for (fp64)."""
        T = len(x)
        t = np.arange(T)
        ids = self.table[b, t // self.page]
        if self.kind in TOP:
            codes, s = quantised(np.asarray(x, np.float64), self.kind)
            self.raw[side][ids, :, t % self.page] = encode(codes, self.kind)
            self.scale[side][ids, :, t % self.page] = s
            return codes * s.astype(np.float64)[..., None]
        raw, value = rounded(x, self.kind)
        self.raw[side][ids, :, t % self.page] = raw
        return value

    def upload(self):
        self.bufs = {n: DB.from_numpy(x) for n, x in self.raw.items()}
        self.sbufs = {n: DB.from_numpy(x) for n, x in self.scale.items()}
        self.tbuf, self.lbuf = ints(self.table), ints(self.lens)
        return self

    def args(self):
        s = [self.sbufs[n] if self.kind in TOP else None for n in "KV"]
        return (self.pages, self.page, self.tbuf, self.ld, self.bufs["K"], self.bufs["V"], *s)

    def download(self):
        return ({n: self.bufs[n].numpy(x.shape, x.dtype) for n, x in self.raw.items()},
                {n: self.sbufs[n].numpy(x.shape, x.dtype) for n, x in self.scale.items()})


def encode(codes, kind):
    """8-bit values as they are stored."""
    if kind == "i8":
        return codes.astype(np.int8)
    n = np.searchsorted(e4m3_values(), np.abs(codes))
    return (n + 128 * np.signbit(codes)).astype(np.uint8)


def decode(raw, kind):
    if kind == "i8":
        return raw.astype(np.float64)
    v = np.append(e4m3_values(), np.nan)
    return np.where(raw & 128, -1.0, 1.0) * v[raw & 127]


# ------------------------------------------------------------------------------ attention

def attention(q, K, V, scale):
    """q: Hq x D; K, V: T x Hk x D.  (o, lse, the largest scale * sum |q k|)."""
    Hq, Hk = len(q), K.shape[1]
    if len(K) == 0:
        return np.zeros_like(q), np.full(Hq, -np.inf), np.zeros(Hq)
    K, V = (np.repeat(x, Hq // Hk, axis=1).transpose(1, 0, 2) for x in (K, V))
    z = scale * np.einsum("hd,htd->ht", q, K)
    m = z.max(-1, keepdims=True)
    e = np.exp(z - m)
    s = e.sum(-1, keepdims=True)
    size = scale * np.einsum("hd,htd->ht", np.abs(q), np.abs(K)).max(-1)
    return np.einsum("ht,htd->hd", e / s, V), (m + np.log(s))[:, 0], size
