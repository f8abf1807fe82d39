"""The groups of sequences that share their first pages: lists that are refused
before a page is read. None needs a GPU."""
import ctypes

import numpy as np
import pytest

import fekv
from fekv import _lib
from fekv.ops import FeError
from test_cpu_8bit_refusals import lib  # noqa: F401  (lib is a fixture)

FAR = 500_000_000
# offsets that leave the three pages of the list although the last one does not
MALFORMED = [[0, FAR, 2 * FAR, 3], [0, 2, 1, 3], [0, 3, 2], [-3, 0, 3], [-FAR, 0, 3], [1, 2, 3],
             [0, -FAR, 3], [0, FAR, 3], [0, 1, FAR, 3, 3], [FAR, 2 * FAR, 3], [0, -1]]


def refused(kv):
    with pytest.raises((FeError, ValueError)) as e:
        fekv.shared_prefixes(kv, [1, 2, 3])
    if isinstance(e.value, FeError):
        assert e.value.status == _lib.FE_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("kv", MALFORMED)
def test_offsets_that_leave_the_list_are_refused(kv):
    refused(kv)


@pytest.mark.parametrize("kv", MALFORMED)
def test_offsets_are_refused_by_the_c_call(kv):
    kv, pages = np.array(kv, np.int32), np.array([1, 2, 3], np.int32)
    off, shared = np.zeros(8, np.int32), np.zeros(8, np.int32)
    n = np.array([7], np.int32)
    L = fekv.load()
    rc = L.fe_kv_shared_prefixes(kv.ctypes.data, pages.ctypes.data, len(kv) - 1, 1,
                                 off.ctypes.data, shared.ctypes.data,
                                 n.ctypes.data_as(ctypes.POINTER(ctypes.c_int)))
    assert rc == _lib.FE_ERR_INVALID_ARGUMENT and n[0] == 0
    assert b"kv" in L.fe_last_error()


@pytest.mark.parametrize("kv", [m for m in MALFORMED if len(m) == 4])
def test_offsets_are_refused_by_prepare(lib, kv, monkeypatch):  # noqa: F811
    """The grouping that SharedPlan.prepare asks for by default."""
    real = fekv.load()
    plan = fekv.SharedPlan(8, 2, 128, 16, 4, 4, True, 3)
    before = lib.count
    for name in ("fe_kv_shared_prefixes", "fe_last_error", "fe_status_string"):
        monkeypatch.setattr(lib, name, getattr(real, name), raising=False)
    with pytest.raises((FeError, ValueError)):
        plan.prepare(np.array([0, 1, 2, 3]), np.array(kv), np.array([1, 2, 3]),
                     np.array([5, 5, 5]))
    assert lib.count == before  # the plan's own call is not reached


def test_lists_without_pages_are_no_group():
    off, shared = fekv.shared_prefixes([0, 0, 2, 2, 3], [1, 2, 3])
    assert off.tolist() == [0, 1, 2, 3, 4] and shared.tolist() == [0, 0, 0, 0]
