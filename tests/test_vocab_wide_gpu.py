"""The losses at sizes whose products take tiles of 64, 128 and 256: every product in every tile and type, with tails in
each extent, rings that run for one, two, three and more pairs of stages, splits, pieces, padding and accumulation.
Values are held to the bounds of test_vocab_precision_gpu."""
import numpy as np
import pytest

from dreamcompiler_amd import hip
from test_vocab_gpu import DT, Loss, ints
from test_vocab_precision_gpu import check

TYPES = [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32")]
# D runs over one to five pairs of 64-k stages, with last pairs whose second half is empty (D % 64 in 1..32), whole or cut.
SHAPES = ([(1030, 8200, d) for d in (40, 72, 104, 136, 200, 264)] + [(520, 4100, d) for d in (24, 65, 128)]
          + [(700, 9001, 104), (1030, 17000, 200), (300, 20000, 900), (1030, 9000, 1030), (2050, 3000, 2049),
             (1500, 9000, 1500), (4100, 300, 2100), (700, 700, 2500), (130, 3800, 2041)])


def plan(N, V, D, K, dtype, grad, extra=64 << 30):
    return hip.linear_loss_plan(DT[dtype], DT[grad], N, V, D, K or 0, extra)


@pytest.mark.parametrize("dtype,grad", TYPES)
def test_shapes_reach_every_product_in_every_tile(dtype, grad):
    plans = [plan(*s, None, dtype, grad) for s in SHAPES]
    for product in range(4):
        assert {p[product] for p in plans} == {64, 128, 256}, (product, plans)
    # 256-wide statistics and G of 1, 2, 3 and 4 pairs of stages; dH and dW whole and in splits
    deep = {(d + 63) // 64 for (_, _, d), p in zip(SHAPES, plans) if p[0] == p[1] == 256}
    assert {1, 2, 3, 4, 5} <= deep
    for t in (64, 128, 256):
        assert any(p[2] == t and p[4] > 1 for p in plans)
    assert any(p[3] == 64 and p[5] > 1 for p in plans) and any(p[5] == 1 for p in plans)


def test_plan_of_few_rows_and_of_small_workspaces():
    assert plan(4, 5000, 64, None, "bf16", "bf16") == (0,) * 8
    assert plan(20, 5000, 64, None, "f32", "f32")[0] == 0 and plan(20, 5000, 64, None, "f32", "f32")[1] > 0
    N, V, D = 300, 5000, 64
    least = max(hip.linear_xent_workspace(hip.F32, N, V, D, b) for b in (0, 1))
    assert plan(N, V, D, None, "f32", "f32", 0)[6:] == (0, 0)
    small, large = plan(N, V, D, None, "f32", "f32", least), plan(N, V, D, None, "f32", "f32", least + (1 << 30))
    assert small[:6] == large[:6] and 256 <= small[7] < large[7] and large[6] >= V and large[7] >= V
    for bad in (dict(dtype=7), dict(grad_type=1, dtype=0), dict(N=0), dict(V=0), dict(D=0), dict(K=-1)):
        a = dict(dtype=0, grad_type=0, N=4, V=9, D=8, K=0, ws_bytes=0)
        with pytest.raises(hip.DreamHipError):
            hip.linear_loss_plan(**{**a, **bad})


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,grad", TYPES)
@pytest.mark.parametrize("K", [None, 5])
@pytest.mark.parametrize("N,V,D", SHAPES)
def test_wide_products(N, V, D, K, dtype, grad):
    """In one piece: 2 GB."""
    c = Loss(N, V, D, dtype, K=K, T=2.0, pad=0.1, seed=D)
    check(c, grad, extra=2 << 30)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,grad", TYPES)
@pytest.mark.parametrize("K", [None, 5])
@pytest.mark.parametrize("N,V,D,ldx", [(1030, 8200, 136, 8), (1030, 17000, 104, 3), (300, 20000, 900, 4), (1030, 9000, 1030, 0)])
def test_wide_products_in_pieces(N, V, D, ldx, K, dtype, grad):
    """Several pieces, the last of them short, with gradients that are added to and rows that have gaps."""
    c = Loss(N, V, D, dtype, K=K, T=2.0, pad=0.3, seed=D, ldx=ldx)
    least = max(c.least(0), c.least(1))
    extra = max(x for x in range(0, 4 * least, least // 16) if plan(N, V, D, K, dtype, grad, least + x)[7] <= V // 2)
    rows = plan(N, V, D, K, dtype, grad, least + extra)[7]
    assert V // 5 < rows < V and V % rows
    check(c, grad, accumulate=True, extra=extra)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,grad", TYPES)
def test_wide_products_of_rows_that_hardly_count(dtype, grad):
    """The tiles are picked for all rows; the extents are those that count: none, one, a tile's edge and one more."""
    N, V, D = 1030, 8200, 72
    for count in (0, 1, 256, 257):
        c = Loss(N, V, D, dtype, seed=count)
        keep = np.zeros(N, bool)
        keep[np.random.default_rng(count).permutation(N)[:count]] = True
        at = c.q.argmax(1)
        c.keep, c.q[~keep] = keep, 0
        c.ids = ints(np.where(keep, at, -1))
        check(c, grad, extra=1 << 30)
