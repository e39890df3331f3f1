"""How attention over a paged cache is split, as its plan tells.  No GPU needed."""
import pytest

from _decoder import TYPE
from dreamcompiler_amd import hip

SIZE = {"f32": 4, "bf16": 2, "i8": 1, "f8": 1}


@pytest.mark.parametrize("kind", SIZE)
@pytest.mark.parametrize("D", [16, 64, 80, 128, 192, 256])
@pytest.mark.parametrize("B,Hk", [(1, 1), (1, 8), (4, 8), (127, 1)])
def test_what_one_work_group_reads_stays_whole(B, Hk, D, kind):
    """256 KB of keys and values, whatever the type and D, and at most 1088 tokens; one token more is split, and only that
    needs a workspace."""
    whole = min((256 << 10) // (2 * D * SIZE[kind]), 1088)
    for n, splits in ((whole // 2, 1), (whole, 1), (whole + 1, 2), (2 * whole, 2)):
        assert (hip.paged_attention_plan(TYPE[kind], B, 4 * Hk, Hk, D, n, 0)[1] > 1) == (splits > 1)
        assert (hip.paged_attention_workspace(TYPE[kind], B, 4 * Hk, Hk, D, n) > 0) == (splits > 1)


@pytest.mark.parametrize("kind", SIZE)
def test_many_sequences_stay_whole_by_tokens(kind):
    for D in (64, 128, 256):
        assert hip.paged_attention_plan(TYPE[kind], 16, 32, 8, D, 1088, 0)[1] == 1
        assert hip.paged_attention_workspace(TYPE[kind], 16, 32, 8, D, 1088) == 0
