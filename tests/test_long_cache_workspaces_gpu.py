"""Scratch memory of the operators over long caches: whatever it holds beyond what a plan wants zeroed, results are the same."""
import pytest
import torch

from test_long_cache_uses_gpu import USES, Use

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", [n for n in USES if n.split()[0] in ("select", "attend", "weigh") and n != "attend alone"])
@pytest.mark.parametrize("poison", [0x7FC00000, -1, 0x3F800000])
def test_workspaces_that_hold_anything(cuda, name, poison):
    use = Use(name, cuda)
    want, space = use.eager(), use.plan.new_workspace()
    assert space.numel() * 4 >= use.plan.plan.workspace_bytes
    space.fill_(poison)
    space[:use.plan.plan.zero_bytes // 4] = 0
    for _ in range(3):
        use.check(use.call(use.fresh(), workspace=space), want)
