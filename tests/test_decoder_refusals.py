"""What the norm of queries and keys, the paged cache and the attention over it refuse, before they touch a
device: no GPU needed.  The addresses are never read."""
import pytest

from dreamcompiler_amd import hip

P, ODD = 1 << 20, (1 << 20) + 8
NAN, INF = float("nan"), float("inf")
BIG = 1 << 40


def raises(match):
    return pytest.raises(hip.DreamHipError, match=match)


def qk_fwd(dt=0, B=2, S=3, Hq=4, Hk=2, D=8, R=8, eps=1e-6, pos=P, table=P, n=9, Q=P, K=P, Qo=P, Ko=P, sq=(96, 32, 8),
           sk=(48, 16, 8), sqo=(96, 32, 8), sko=(48, 16, 8)):
    hip.qk_norm_rope_fwd(dt, B, S, Hq, Hk, D, R, False, eps, pos, table, n, Q, sq, K, sk, None, None, Qo, sqo, Ko, sko)


def qk_bwd(dt=0, B=2, S=3, Hq=4, Hk=2, D=8, R=8, eps=1e-6, pos=P, table=P, n=9, Q=P, K=P, dQo=P, dKo=P, dQ=P, dK=P,
           sq=(96, 32, 8), sk=(48, 16, 8), sdqo=(96, 32, 8), sdko=(48, 16, 8), sdq=(96, 32, 8), sdk=(48, 16, 8), dout=0, gt=0,
           dgq=None, dgk=None, ws=P, size=BIG):
    hip.qk_norm_rope_bwd(dt, B, S, Hq, Hk, D, R, False, eps, pos, table, n, Q, sq, K, sk, None, None, dout, dQo, sdqo, dKo,
                         sdko, gt, dQ, sdq, dK, sdk, dgq, dgk, False, ws, size)


def write(dt=0, ct=3, B=2, N=5, Hk=2, D=32, K=P, sk=(64, 32), V=P, sv=(64, 32), first=P, len_=P, pages=4, page=16, table=P,
          ld=2, Kc=P, Vc=P, Ks=P, Vs=P):
    hip.kv_cache_write(dt, ct, B, N, Hk, D, K, sk, V, sv, first, len_, pages, page, table, ld, Kc, Vc, Ks, Vs)


def read(dt=0, ct=3, B=2, N=5, Hk=2, D=32, K=P, sk=(64, 32), V=P, sv=(64, 32), first=P, len_=P, pages=4, page=16, table=P,
         ld=2, Kc=P, Vc=P, Ks=P, Vs=P):
    hip.kv_cache_read(dt, ct, B, N, Hk, D, K, sk, V, sv, first, len_, pages, page, table, ld, Kc, Vc, Ks, Vs)


def attend(dt=0, ct=3, B=2, Hq=4, Hk=2, D=32, scale=1.0, window=0, Q=P, sq=(128, 32), len_=P, max_len=32, pages=4, page=16,
           table=P, ld=2, Kc=P, Vc=P, Ks=P, Vs=P, O=P, so=(128, 32), ws=P, size=BIG):
    hip.paged_attention(dt, ct, B, Hq, Hk, D, scale, window, Q, sq, len_, max_len, pages, page, table, ld, Kc, Vc, Ks, Vs, O,
                        so, None, ws, size)


QK, CACHE = [qk_fwd, qk_bwd], [write, read, attend]


@pytest.mark.parametrize("f", QK + CACHE)
def test_types(f):
    for dt in (-1, 2, 3, 4, 7):
        with raises("dtype"):
            f(dt=dt)


@pytest.mark.parametrize("f", CACHE)
def test_cache_types(f):
    for dt, ct in ((0, 1), (1, 0), (0, 2), (0, 5), (1, -1)):
        with raises("cache_type"):
            f(dt=dt, ct=ct)


@pytest.mark.parametrize("f", QK)
def test_qk_shapes(f):
    for bad in (dict(B=-1), dict(S=-1), dict(Hq=-1), dict(Hk=65537), dict(D=0), dict(D=1025), dict(B=2 ** 16, S=2 ** 15)):
        with raises("shape"):
            f(**bad)
    for R in (-2, 3, 10):
        with raises("R="):
            f(R=R)
    for eps in (0.0, -1.0, 1e-39, NAN, INF):
        with raises("eps"):
            f(eps=eps)
    for bad in (dict(table=None), dict(n=0), dict(pos=None, n=2), dict(R=0, n=0)):
        with raises("no table"):
            f(**bad)


@pytest.mark.parametrize("f,names", [(qk_fwd, "sq sk sqo sko"), (qk_bwd, "sq sk sdqo sdko sdq sdk")])
def test_qk_strides(f, names):
    for n in names.split():
        with raises("null strides"):
            f(**{n: None})
        for s in ((96, 32, -8), (1 << 46, 32, 8), (1 << 62, 32, 8), (-1, 32, 8)):
            with raises("strides"):
                f(**{n: s})
    for n in ("sqo sko" if f is qk_fwd else "sdq sdk").split():
        for s in ((96, 32, 7), (96, 8, 8), (0, 32, 8), (33, 32, 8), (96, 0, 8)):   # rows over each other
            with raises("strides"):
                f(**{n: s})


@pytest.mark.parametrize("f,names", [(qk_fwd, "Q K Qo Ko"), (qk_bwd, "Q K dQo dKo dQ dK ws"), (write, "K V len_ table Kc Vc Ks Vs"),
                                     (read, "K V len_ table Kc Vc Ks Vs"), (attend, "Q len_ O table Kc Vc Ks Vs")])
def test_null_pointers(f, names):
    for n in names.split():
        with raises("null"):
            f(**{n: None})
    if f is attend:
        with raises("null"):
            f(B=1, ld=8192, max_len=131072, ws=None)


def test_qk_gradient_types_and_workspace():
    for bad in (dict(dout=1), dict(gt=1), dict(dt=1, dout=3), dict(dt=1, gt=2)):
        with raises("dout_type and grad_type"):
            qk_bwd(**bad)
    assert hip.qk_norm_rope_bwd_workspace(0) == 0 and hip.qk_norm_rope_bwd_workspace(2000) == 0
    for D in (8, 128, 1024):
        need = hip.qk_norm_rope_bwd_workspace(D)
        big = (1 << 20, 1 << 15, 1 << 11)
        a = dict(D=D, sq=big, sk=big, sdqo=big, sdko=big, sdq=big, sdk=big)
        with raises("workspace of"):
            qk_bwd(size=need - 1, **a)
        with raises("aligned"):
            qk_bwd(ws=ODD, **a)


def test_weights_gradients_apart():
    for d in (0, 4, 28, -28):
        with raises("overlap"):
            qk_bwd(dgq=P, dgk=P + d)


def test_tables():
    for bad in ((-1, 8, 1e4), (4, -2, 1e4), (4, 7, 1e4), (4, 2048, 1e4)):
        with raises("shape"):
            hip.rope_table(*bad, P)
    for base in (0.0, -1.0, NAN, INF):
        with raises("base"):
            hip.rope_table(4, 8, base, P)
    with raises("null"):
        hip.rope_table(4, 8, 1e4, None)


@pytest.mark.parametrize("f", CACHE)
def test_cache_shapes(f):
    for bad in (dict(B=-1), dict(B=65536), dict(Hk=0), dict(Hk=65536), dict(D=0), dict(D=8), dict(D=40), dict(D=272)):
        with raises("shape"):
            f(**bad)
    for page in (0, -16, 8, 24, 8192):
        with raises("page="):
            f(page=page)
    for bad in (dict(pages=0), dict(ld=0), dict(pages=2 ** 31 - 1, page=4096, D=256, Hk=64)):
        with raises("pages="):
            f(**bad)
    for n in ("Kc", "Vc", "Ks", "Vs"):
        with raises("aligned"):
            f(**{n: ODD})


@pytest.mark.parametrize("f", [write, read])
def test_cache_rows(f):
    for bad in (dict(N=-1), dict(N=2 ** 29 + 1), dict(N=2 ** 31 - 1), dict(first=None)):
        with raises("tokens"):
            f(**bad)
    for n in ("sk", "sv"):
        with raises("null strides"):
            f(**{n: None})
        for s in ((64, -32), (1 << 46, 32), (-1, 32)):
            with raises("strides"):
                f(**{n: s})
    if f is read:
        for s in ((64, 31), (32, 32), (63, 32), (0, 32), (64, 0)):
            with raises("strides"):
                f(sk=s)


def test_attention_arguments():
    for bad in (dict(Hq=0), dict(Hq=3), dict(Hq=-4), dict(Hq=131072)):
        with raises("Hq="):
            attend(**bad)
    for s in (0.0, -1.0, NAN, INF):
        with raises("scale"):
            attend(scale=s)
    with raises("shape"):
        attend(B=65535, Hq=128, sq=(128 * 32, 32), so=(128 * 32, 32))
    for bad in (dict(window=-1), dict(max_len=-1), dict(max_len=33), dict(ld=2 ** 22, max_len=2 ** 25 + 1)):
        with raises("max_len"):
            attend(**bad)
    for n in ("sq", "so"):
        with raises("null strides"):
            attend(**{n: None})
        with raises("strides"):
            attend(**{n: (128, -32)})
    for s in ((128, 31), (0, 32), (33, 32)):
        with raises("strides"):
            attend(so=s)
    need = hip.paged_attention_workspace(3, 1, 4, 2, 32, 131072)
    assert need > 0
    with raises("workspace of"):
        attend(B=1, ld=8192, max_len=131072, size=need - 1)
    with raises("aligned"):
        attend(B=1, ld=8192, max_len=131072, ws=ODD)
    assert hip.paged_attention_workspace(3, 1, 4, 2, 32, 16) == 0
    assert hip.paged_attention_workspace(3, 0, 4, 2, 32, 1000) == 0


def test_plans_fit_their_workspaces():
    """For lengths, windows and shapes of all sizes: the chunks cover what is seen, a work-group's lanes hold a
    chunk's pages, the launch holds the chunks, and the query's workspace has room for the partial results of every window."""
    for ct in (0, 1, 3, 4):
        for B, Hq, Hk, D in ((1, 1, 1, 16), (1, 32, 8, 128), (3, 12, 3, 80), (16, 16, 8, 256), (64, 64, 8, 128), (500, 40, 2, 64),
                             (4096, 8, 8, 32), (65535, 64, 1, 256)):
            for max_len in (0, 1, 31, 128, 512, 513, 1088, 1089, 2047, 5000, 40000, 131072, 2 ** 20, 2 ** 25):
                room = hip.paged_attention_workspace(ct, B, Hq, Hk, D, max_len)
                for window in (0, 1, 97, 512, 1000, 1057, 1058, 3000, 33333, 2 ** 31 - 1):
                    chunk, splits, waves, groups = hip.paged_attention_plan(ct, B, Hq, Hk, D, max_len, window)
                    seen = min(max_len, window + 31) if window else max_len
                    assert chunk % 128 == 0 and 128 <= chunk <= 2048 and 1 <= splits <= 65535
                    assert chunk * splits >= seen and waves in (4, 8)
                    assert groups == (-(-(Hq // Hk) // 32) if Hq // Hk > 16 else 1)
                    need = splits * B * Hq * (D + 2) * 4 if splits > 1 else 0
                    assert need <= room, (ct, B, Hq, Hk, D, max_len, window)
    for bad in (dict(B=0), dict(Hq=3), dict(D=300), dict(max_len=-1), dict(window=-1), dict(max_len=2 ** 25 + 1)):
        a = {**dict(cache_type=3, B=2, Hq=4, Hk=2, D=32, max_len=100, window=0), **bad}
        with raises("shape"):
            hip.paged_attention_plan(**a)
