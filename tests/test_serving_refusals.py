"""Refusals of the serving operators' descriptors at the ends of their ints (CPU: all
before any GPU call)."""
import pytest

import hipgemm_amd as hg
from hipgemm_amd import serving
from test_torch_serving import INVALID, _moe_desc, _w4_desc

#: The largest group sizes: K + group_size - 1 is past an int.
HUGE = (2 ** 31 - 32, 2 ** 31 - 64)


@pytest.mark.parametrize("group", HUGE)
@pytest.mark.parametrize("lds", [0, -1, -(1 << 40)])
def test_groups_of_a_whole_row_need_a_scale(group, lds):
    assert serving.w4_gemm_raw(_w4_desc(group_size=group, lds=lds)) == INVALID
    bad = dict(lds=lds, expert_s=128)
    kw = dict(format=0, scale_type=1, group_size=group)
    assert serving.moe_experts_raw(_moe_desc(w13=bad, **kw)) == INVALID
    assert serving.moe_experts_raw(_moe_desc(w2=bad, **kw)) == INVALID


@pytest.mark.parametrize("group", HUGE)
def test_groups_of_a_whole_row_are_taken(group):
    assert hg.w4_select(_w4_desc(group_size=group, lds=1))[0] == "vectors"
