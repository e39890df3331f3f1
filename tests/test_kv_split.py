"""How the cache's reads and writes are split over a wave's lanes: the header's own functions, compiled for the
host.  No GPU needed."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def split(tmp_path_factory):
    d = tmp_path_factory.mktemp("split")
    src, lib = d / "s.cpp", d / "s.so"
    src.write_text('#include "dh_kv_split.hpp"\n'
                   'extern "C" void split(int N, int Hk, int places, int ahead, long long* out) {\n'
                   '  const dh::Split s = dh::split_tokens(N, Hk, places, ahead);\n'
                   '  const long long v[] = {s.tokens, s.log_heads, s.blocks, s.each, s.per, s.units, s.many};\n'
                   '  for (int i = 0; i < 7; ++i) out[i] = v[i];\n'
                   '}\n'
                   'extern "C" int first_token(int sub, int log_heads) { return dh::first_token(sub, log_heads); }\n'
                   'extern "C" int rounds(int t, int side, int ahead) { return dh::rounds_of(t, side, ahead); }\n')
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "dreamcompiler_amd", "csrc"),
                    str(src), "-o", str(lib)], check=True)
    f = ctypes.CDLL(str(lib))

    def call(*a):
        out = (ctypes.c_longlong * 7)()
        f.split(*a, out)
        return dict(zip("tokens log_heads blocks each per units many".split(), out))
    return call, f.first_token, f.rounds


TOKENS = [1, 2, 3, 15, 64, 1000, 24575, 24576, 52001, 74000, 100000, 400000, 5000000, 1 << 29]


@pytest.mark.parametrize("ahead", [1, 2])
@pytest.mark.parametrize("places", [1, 2, 4, 8, 16])
@pytest.mark.parametrize("Hk", [1, 2, 3, 4, 5, 8, 9, 16, 40, 65535])
def test_rounds_cover_each_head_of_each_token_once(split, Hk, places, ahead):
    """A wave that has several tokens at once makes no more rounds than its tokens need, and its places cover
    every head of every token once, one head of keys (a token's places are 2^0) included."""
    of, first, rounds = split
    for N in TOKENS:
        u = of(N, Hk, places, ahead)
        assert 1 <= u["tokens"] <= 64 and u["units"] < 1 << 31
        groups = u["units"] // u["per"]
        assert groups * u["tokens"] >= N and u["per"] * u["each"] >= u["blocks"]
        if not u["many"]:
            assert u["blocks"] * places * ahead >= Hk
            continue
        heads = 1 << u["log_heads"]
        side = places // heads
        n = rounds(u["tokens"], side, ahead)
        assert heads >= Hk and u["tokens"] % side == 0
        assert (n - 1) * ahead * side < u["tokens"] <= n * ahead * side
        seen = [(sub % heads, t) for sub in range(places) for k in range(n) for a in range(ahead)
                for t in [first(sub, u["log_heads"]) + (k * ahead + a) * side] if t < u["tokens"]]
        assert sorted(seen) == [(h, t) for h in range(heads) for t in range(u["tokens"])]


def test_sizes_that_once_made_a_round_for_nothing(split):
    """8 heads of 32 bf16 (16 places), and 2 heads of 128 bf16 (4 places) over 100000 tokens, 4 a wave: one round."""
    of, _, rounds = split
    for N in (1, 1000, 24575):
        u = of(N, 8, 16, 2)
        assert u["many"] and rounds(u["tokens"], 16 >> u["log_heads"], 2) == 1
    u = of(100000, 2, 4, 2)
    assert (u["tokens"], rounds(u["tokens"], 4 >> u["log_heads"], 2)) == (4, 1)
