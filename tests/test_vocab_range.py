"""The address ranges that the vocabulary products give their loads end with the operand: the header's own functions,
compiled for the host.  No GPU needed."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from test_vocab_gpu import DT, Loss, run_loss
from _gpu import DB
from dreamcompiler_amd import hip

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def ranges(tmp_path_factory):
    d = tmp_path_factory.mktemp("range")
    src, lib = d / "r.cpp", d / "r.so"
    src.write_text('#include "dh_vocab_range.hpp"\n'
                   'extern "C" unsigned bytes(int r, int ld, int e, int t0) { return dh::range_bytes(r, ld, e, t0); }\n')
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "dreamcompiler_amd", "csrc"),
                    str(src), "-o", str(lib)], check=True)
    f = ctypes.CDLL(str(lib)).bytes
    f.restype = ctypes.c_uint
    return f


@pytest.mark.parametrize("T,BK", [(64, 64), (128, 32), (256, 32)])
@pytest.mark.parametrize("K,D,ld", [(1, 8, 8), (33, 72, 4096), (64, 264, 272), (100, 1000, 1000), (4097, 200, 456),
                                    (256, 8, 1 << 22)])
def test_rows_of_k_end_with_the_last_row(ranges, T, BK, K, D, ld):
    """[k][column], K x D in rows of ld: the buffer holds (K - 1) ld + D values and no more.  Every stage of every
    tile reaches no further, and reaches each of its own values."""
    end = 2 * ((K - 1) * ld + D)
    for kt in {0, max(0, (K - 1) // BK - 1), (K - 1) // BK}:
        rows = min(K - kt * BK, BK)
        for t0 in {0, (D - 1) // T * T}:
            base = 2 * (kt * BK * ld + t0)
            n = ranges(rows, ld, D, t0)
            assert base + n <= end
            last = 2 * ((rows - 1) * ld + min(T, D - t0))   # behind the tile's last value
            assert n >= last


@pytest.mark.parametrize("rows,K,ld", [(1, 8, 8), (256, 1000, 1 << 22), (17, 72, 4096), (64, 264, 272)])
def test_rows_of_columns_end_with_the_last_column(ranges, rows, K, ld):
    """[row][k]: the last row's K values, not its ld; 256 rows of 2^22 stay within 32 bits."""
    assert ranges(rows, ld, K, 0) == 2 * ((rows - 1) * ld + K)


def test_nothing_left(ranges):
    assert ranges(0, 64, 64, 0) == ranges(-5, 64, 64, 0) == 0


def test_odd_extents_keep_their_last_value(ranges):
    """Ranges are checked by 4-byte words: an odd extent keeps the word that its last value lies in."""
    for e in (1, 7, 9, 33, 1001):
        n = ranges(5, 2048, e, 0)
        assert n % 16 == 0 and n >= 2 * (4 * 2048 + e)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [None, 4])
@pytest.mark.parametrize("N,V,D,wide", [(70, 300, 40, 64), (300, 1025, 72, 256), (9, 700, 104, 1024), (1030, 8200, 72, 80)])
def test_a_table_inside_a_wider_matrix(N, V, D, wide, K):
    """W is the right-hand columns of a matrix: its last row ends with the buffer."""
    c = Loss(N, V, D, "bf16", K=K)
    r = np.random.default_rng(0)
    raw = r.integers(0, 1 << 16, (V, wide)).astype(np.uint16)
    raw[:, wide - D:] = c.Wb.numpy((V, D), np.uint16)
    whole = DB.from_numpy(raw)
    base, ld = whole.ptr + 2 * (wide - D), wide
    size = max(c.least(0), c.least(1)) + (1 << 20)

    def run(W, ldw):
        ws = DB(size)
        loss, lse = DB.empty((N,), np.float32), DB.empty((N,), np.float32)
        dH, dW = DB.empty((N, D), np.uint16), DB.empty((V, D), np.uint16)
        head = list(c.head())
        at = 7 if K is None else 8
        head[at:at + 2] = [W, ldw]
        (hip.linear_xent_fwd if K is None else hip.linear_distill_fwd)(*head, loss, lse, ws, size)
        (hip.linear_xent_bwd if K is None else hip.linear_distill_bwd)(
            *head, lse, c.dlb, dH, D, False, dW, D, False, DT["bf16"], ws, size)
        return [x.numpy() for x in (loss, lse, dH, dW)]

    for a, b in zip(run(c.Wb, D), run(base, ld)):
        assert np.array_equal(a, b)
    run_loss(c)
