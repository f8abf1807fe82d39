"""Budgets whose entries' indexes would pass 31 bits in a kernel, and addresses that a
kernel could not read, are refused before anything is launched. None needs a GPU."""
import pytest

import fekv
from fekv import _lib
from test_cpu_long_prompt_refusals import P, compact_c, select_c


@pytest.mark.parametrize("call", [select_c, compact_c])
@pytest.mark.parametrize("budget", [(1 << 30) + 1, (1 << 31) - 256, (1 << 31) - 1])
def test_budgets_above_2_30(call, budget):
    assert call(budget=budget) == _lib.FE_ERR_CAPACITY
    assert b"budget" in fekv.load().fe_last_error()
    assert call(batch=0, budget=1 << 30) == _lib.FE_OK


@pytest.mark.parametrize("call,kw", [(select_c, dict(kept=P + 2)), (compact_c, dict(kept=P + 2)),
                                     (compact_c, dict(scores=P + 2)),
                                     (compact_c, dict(scores=P + 1))])
def test_lists_and_scores_between_their_elements(call, kw):
    assert call(**kw) == _lib.FE_ERR_INVALID_ARGUMENT
    assert b"aligned" in fekv.load().fe_last_error()
