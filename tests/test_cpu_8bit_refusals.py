"""Arguments that the 8-bit cache's calls refuse before anything is launched,
beside those of test_cpu_kv8.py. None needs a GPU."""
import pytest

import fekv
from fekv import _lib
from test_cpu_kv8 import gather_args


@pytest.mark.parametrize("cs", [8, 24, 40, 17])
def test_gather_refuses_slots_without_a_scale_of_their_own(cs):
    """One scale row per 16 slots: a pool's last slots would read past them."""
    assert fekv.load().fe_kv8_gather(*gather_args(cs=cs)) == _lib.FE_ERR_INVALID_ARGUMENT
    assert b"cache_slots" in fekv.load().fe_last_error()
