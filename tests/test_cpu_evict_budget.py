"""Budgets whose entries' indexes would pass 31 bits in a kernel are refused before
anything is launched. None needs a GPU."""
import pytest

import fekv
from fekv import _lib
from test_cpu_long_prompt_refusals import compact_c, select_c


@pytest.mark.parametrize("call", [select_c, compact_c])
@pytest.mark.parametrize("budget", [(1 << 30) + 1, (1 << 31) - 256, (1 << 31) - 1])
def test_budgets_above_2_30(call, budget):
    assert call(budget=budget) == _lib.FE_ERR_CAPACITY
    assert b"budget" in fekv.load().fe_last_error()
    assert call(batch=0, budget=1 << 30) == _lib.FE_OK
