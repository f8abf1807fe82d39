"""Offsets of a step that leave its page list in the middle: the planners refuse them
before they read a page behind the list. None needs a GPU."""
import numpy as np
import pytest

import fekv
from fekv import _lib
from fekv.ops import FeError
from test_cpu_long_plan import Host

HOSTS = {
    "plan": lambda: fekv.HostPlan(8, 2, 128, 16, 4, 64, True, 9),
    "kv8": lambda: fekv.HostKv8Plan(8, 2, 128, 16, 4, 64, True, 9),
    "shared": lambda: Host(8, 2, 128, 16, 4, 64, 9),
    "scored": lambda: Host(8, 2, 128, 16, 4, 64, 9, True, 4096),
}


@pytest.mark.parametrize("kv", [[0, 40, 3], [0, 2, 40, 3], [0, 40, 41, 3]])
@pytest.mark.parametrize("kind", HOSTS)
def test_offsets_are_checked_before_pages(kind, kv):
    """The list has three pages. What lies behind them here is no page id at all:
    a planner that looks there complains of it and not of the offsets."""
    behind = np.full(64, 1 << 20, np.int32)
    behind[:3] = [1, 2, 3]
    n = len(kv) - 1
    plan = HOSTS[kind]()
    with pytest.raises(FeError, match="own at least one page") as e:
        if kind == "shared":
            plan.prepare(np.arange(n + 1), kv, behind, [5] * n, groups=([0, n], [0]))
        else:
            plan.prepare(np.arange(n + 1), np.array(kv), behind, np.array([5] * n))
    assert e.value.status == _lib.FE_ERR_INVALID_ARGUMENT
