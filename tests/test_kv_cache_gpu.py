"""A paged key-value cache: what a write leaves in it and what a read takes from it, against the definition in
64 bits, to the last bit: 8-bit values are those of the exact quotient, a read rounds value * scale
to fp32 and then to its type."""
import numpy as np
import pytest

from _decoder import TOP, TYPE, Cache, Strided, decode, encode, ints, quantised, rounded
from _gpu import DB
from dreamcompiler_amd import hip

KINDS = [("f32", "f32"), ("f32", "i8"), ("f32", "f8"), ("bf16", "bf16"), ("bf16", "i8"), ("bf16", "f8")]


def starts(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def read_back(value, scale, kind, dtype):
    """What a read gives for stored values: fp32 product, then the type."""
    x = value.astype(np.float32)
    if kind in TOP:
        x = x * scale[..., None]
    return rounded(x, dtype)[1] if dtype == "bf16" else x.astype(np.float64)


def run(dtype, kind, lens, new, Hk, D, page, pad=0, order=(0, 1), ones=False, tail=2, seed=0, values=None, spoil=()):
    """Writes each sequence's last new[b] tokens, looks at the whole cache, and reads all back."""
    r = np.random.default_rng(seed)
    c = Cache(kind, lens, Hk, D, page, seed)
    for b, i, v in spoil:
        c.table[b, i] = v
    c.upload()
    first = starts(new)
    N = int(first[-1])
    lead = 0 if ones else 1            # a row before the first sequence's
    rows = N + lead + (0 if ones else tail)
    if not ones:
        first = first + lead
    x = [r.standard_normal((rows, Hk, D)) * np.exp2(r.integers(-6, 7, (rows, Hk, 1))) for _ in "KV"]
    if values is not None:
        x = [values(r, (rows, Hk, D)) for _ in "KV"]
    K, V = (Strided(y, dtype, order, pad) for y in x)
    fb = None if ones else ints(first)
    hip.kv_cache_write(TYPE[dtype], TYPE[kind], len(lens), rows, Hk, D, K, K.strides, V, V.strides, fb, c.lbuf, *c.args())
    raw, scale = c.download()
    want_raw, want_scale = ({n: y.copy() for n, y in d.items()} for d in (c.raw, c.scale))
    stands = {n: np.zeros((len(lens), max(max(lens, default=0), 1), Hk, D)) for n in "KV"}
    for n, y in (("K", K), ("V", V)):
        for b, m in enumerate(new):
            for i in range(m):
                t = lens[b] - m + i
                if t < 0 or t // page >= c.ld or not 0 <= c.table[b, t // page] < c.pages:
                    continue
                at = (c.table[b, t // page], slice(None), t % page)
                row = y.value[first[b] + i]
                if kind in TOP:
                    codes, s = quantised(row, kind)
                    want_raw[n][at], want_scale[n][at] = encode(codes, kind), s
                else:
                    want_raw[n][at] = rounded(row, kind)[0]
    for n in "KV":
        if kind in TOP:
            assert np.array_equal(scale[n], want_scale[n], equal_nan=True)
            held = ~np.isnan(want_scale[n])
            # zero has two codes, which stand for the same
            assert np.array_equal(decode(raw[n], kind)[held], decode(want_raw[n], kind)[held])
            untouched = want_raw[n] == c.raw[n]
            assert np.array_equal(raw[n][untouched & ~held[..., None]], want_raw[n][untouched & ~held[..., None]])
        else:
            assert np.array_equal(raw[n].view(np.uint8), want_raw[n].view(np.uint8))
    # all of every sequence, behind a row that is of none and before two more
    every = starts([max(m, 0) for m in lens]) + 1
    M = int(every[-1]) + 2
    out = [Strided(np.full((M, Hk, D), 7.0), dtype, order, pad) for _ in "KV"]
    hip.kv_cache_read(TYPE[dtype], TYPE[kind], len(lens), M, Hk, D, out[0], out[0].strides, out[1], out[1].strides,
                      ints(every), c.lbuf, *c.args())
    for n, o in zip("KV", out):
        want = np.full((M, Hk, D), 7.0)
        for b, m in enumerate(lens):
            for t in range(m):
                want[every[b] + t] = 0.0
                if t // page < c.ld and 0 <= c.table[b, t // page] < c.pages:
                    at = (c.table[b, t // page], slice(None), t % page)
                    v = raw[n][at]
                    v = decode(v, kind) if kind in TOP else (v if kind == "f32" else
                                                             (v.astype(np.uint32) << 16).view(np.float32))
                    want[every[b] + t] = read_back(v, scale[n][at] if kind in TOP else None, kind, dtype)
        got = o.get()
        assert np.array_equal(got, want, equal_nan=True)
    return c, raw, scale


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("Hk,D,page", [(1, 16, 16), (2, 64, 16), (3, 80, 32), (8, 128, 64), (1, 256, 128), (5, 96, 16),
                                       (2, 112, 4096)])
def test_write_and_read(Hk, D, page, dtype, kind):
    run(dtype, kind, [1, 40, 0, 17, 130], [1, 23, 0, 17, 1], Hk, D, page)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
def test_one_token_each(dtype, kind):
    run(dtype, kind, [1, 16, 17, 33, 100], [1] * 5, 4, 128, 16, ones=True)
    run(dtype, kind, [5, 0, -3], [1] * 3, 2, 32, 16, ones=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("pad,order", [(0, (1, 0)), (1, (0, 1)), (8, (1, 0)), (16, (0, 1)), (3, (1, 0))])
def test_strides(pad, order, dtype, kind):
    run(dtype, kind, [9, 30], [4, 30], 3, 64, 16, pad=pad, order=order)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
def test_pages_that_hold_nothing(dtype, kind):
    """Table entries outside the pages, and more new tokens than a sequence holds."""
    run(dtype, kind, [70, 40], [70, 40], 2, 48, 16, spoil=[(0, 1, -1), (0, 3, 2 ** 31 - 1), (1, 0, 10 ** 6), (1, 2, -2 ** 31)])
    run(dtype, kind, [10, 3, 20], [15, 8, 20], 2, 48, 16)


def borders(r, shape):
    """Rows whose quotients lie on the borders between two values and right beside them."""
    x = np.zeros(shape, np.float32)
    top = np.exp2(r.integers(-30, 30, shape[:-1])).astype(np.float32) * (1 + r.random(shape[:-1])).astype(np.float32)
    s = (top / 127.0).astype(np.float32)
    half = (r.integers(0, 127, shape) + 0.5).astype(np.float32)
    x[:] = s[..., None] * half
    way = r.random(shape)
    x = np.nextafter(x, np.where(way < 0.33, np.inf, np.where(way < 0.67, -np.inf, x)).astype(np.float32))
    x *= np.where(r.random(shape) < 0.5, 1, -1)
    x[..., 0] = top
    return x


def powers(r, shape):
    """Rows whose largest value is the type's top times a power of two: exact quotients, ties among them."""
    x = r.integers(-254, 255, shape) / 2.0
    x[..., 0] = 127.0
    return x * np.exp2(r.integers(-40, 40, shape[:-1]))[..., None]


def eighths(r, shape):
    """The same for e4m3: 448 and values half way between two."""
    x = r.integers(-256, 257, shape) * np.exp2(r.integers(-12, 1, shape).astype(np.float64))
    x[..., 0] = 448.0
    return x * np.exp2(r.integers(-40, 40, shape[:-1]))[..., None]


def tiny(r, shape):
    """Down to subnormal scales, zero among them."""
    x = r.standard_normal(shape) * np.exp2(r.integers(-150, -100, shape[:-1]))[..., None]
    return x.astype(np.float32)


def huge(r, shape):
    return (r.standard_normal(shape) * 2.0 ** 125).clip(-3e38, 3e38)


def broken(r, shape):
    """Rows with an infinity or a NaN among others."""
    x = r.standard_normal(shape)
    x[::3, :, 2] = np.inf
    x[1::5, :, 5] = np.nan
    x[4::7, :, 7] = -np.inf
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", [("f32", "i8"), ("f32", "f8"), ("bf16", "i8"), ("bf16", "f8")])
@pytest.mark.parametrize("values", [borders, powers, eighths, tiny, huge, broken], ids=lambda f: f.__name__)
def test_roundings(values, dtype, kind):
    with np.errstate(invalid="ignore", over="ignore"):
        run(dtype, kind, [90, 61], [90, 61], 2, 64, 16, values=values)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
def test_many_tokens(dtype, kind):
    """More rows than waves of a launch."""
    run(dtype, kind, [2100, 1, 900], [2100, 1, 450], 6, 32, 32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("Hk,D", [(1, 16), (2, 80), (3, 32), (5, 256)])
def test_many_sequences(Hk, D, dtype, kind):
    """More sequences than lanes, empty ones among them, beside few heads (several tokens a wave) and many."""
    lens = [(7 * b) % 23 for b in range(150)]
    run(dtype, kind, lens, [n if b % 3 else n // 2 for b, n in enumerate(lens)], Hk, D, 16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("Hk,D,T", [(1, 32, 60000), (2, 64, 52001), (9, 16, 51000)])
def test_long(Hk, D, T, dtype, kind):
    """Several tokens a wave, by turns of four waves; all of a sequence written, and read back."""
    r = np.random.default_rng(4)
    page = 64
    c = Cache(kind, [T], Hk, D, page).upload()
    K, V = (Strided(r.standard_normal((T, Hk, D)), dtype) for _ in "KV")
    first = ints([0, T])
    hip.kv_cache_write(TYPE[dtype], TYPE[kind], 1, T, Hk, D, K, K.strides, V, V.strides, first, c.lbuf, *c.args())
    out = [Strided(np.zeros((T, Hk, D)), dtype) for _ in "KV"]
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
            assert np.array_equal(raw[n][at].view(np.uint8), rounded(x.value, kind)[0].view(np.uint8))
        assert np.array_equal(o.get(), read_back(codes, s, kind, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("first", [[5, 3, 9, 9], [-7, 4, 2, 12], [0, 2 ** 31 - 1, 3, 6], [0, 0, 0, 0], [9, 9, 9, 9]])
def test_beginnings_that_do_not_rise(first):
    """What no caller means: nothing is read or written out of place, and rows of no sequence stay."""
    Hk, D, N = 2, 32, 8
    c = Cache("bf16", [20, 20, 20], Hk, D, 16).upload()
    K = Strided(np.ones((N, Hk, D)), "bf16")
    hip.kv_cache_write(hip.BF16, hip.BF16, 3, N, Hk, D, K, K.strides, K, K.strides, ints(first), c.lbuf, *c.args())
    out = Strided(np.full((N, Hk, D), 7.0), "bf16")
    hip.kv_cache_read(hip.BF16, hip.BF16, 3, N, Hk, D, out, out.strides, out, out.strides, ints(first), c.lbuf, *c.args())
    got, raw = out.get(), c.download()[0]["K"]
    assert (np.isnan(got) | (got == 0) | (got == 1) | (got == 7)).all()
    assert ((raw == 0x7FC0) | (raw == 0x3F80)).all()
    if first in ([0, 0, 0, 0], [9, 9, 9, 9]):
        assert (got == 7).all() and (raw == 0x7FC0).all()


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Places whose offsets pass 2^32 values and 2^32 rows' bytes."""
    Hk, D, page, pages = 8, 256, 4096, 700          # 5.9e9 values
    Kc, Vc = DB(pages * Hk * page * D), DB(pages * Hk * page * D)
    Ks, Vs = (DB(pages * Hk * page * 4) for _ in "KV")
    r = np.random.default_rng(0)
    lens = [4097, 5]
    table = np.array([[699, 600], [3, -1]], np.int32)
    held = (pages, page, ints(table), 2, Kc, Vc, Ks, Vs)
    K, V = (Strided(r.standard_normal((7, Hk, D)), "f32") for _ in "KV")
    first, len_ = ints([0, 2, 7]), ints(lens)
    hip.kv_cache_write(hip.F32, hip.I8, 2, 7, Hk, D, K, K.strides, V, V.strides, first, len_, *held)
    out = [Strided(np.zeros((7, Hk, D)), "f32") for _ in "KV"]
    hip.kv_cache_read(hip.F32, hip.I8, 2, 7, Hk, D, out[0], out[0].strides, out[1], out[1].strides, first, len_, *held)
    for x, o in ((K, out[0]), (V, out[1])):
        codes, s = quantised(x.value, "i8")
        assert np.array_equal(o.get(), (codes.astype(np.float32) * s[..., None]).astype(np.float64))
