"""The groups of sequences that share their first pages: lists that are refused
before a page is read, and which neighbours form a group. None needs a GPU."""
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


# ---------------------------------------------------------------------------
# which neighbours form a group
# ---------------------------------------------------------------------------

def tables_of(edges, extra=1):
    """Page lists whose neighbours b - 1 and b have edges[b - 1] pages in common and
    then differ."""
    tables, fresh = [], iter(range(10 ** 6))
    first = [next(fresh) for _ in range(max(edges, default=0) + extra)]
    tables.append(first)
    for e in edges:
        t = tables[-1][:e]
        t += [next(fresh) for _ in range(max(edges) + extra - len(t))]
        tables.append(t)
    return tables


def groups_of(tables, least=1):
    kv = np.cumsum([0] + [len(t) for t in tables])
    off, shared = fekv.shared_prefixes(kv, np.concatenate(tables), least)
    return off.tolist(), shared.tolist()


def saved(off, shared):
    return sum((e - a - 1) * n for a, e, n in zip(off, off[1:], shared))


def most(edges, least=1):
    """The best cut by trying every one."""
    n, best = len(edges) + 1, 0
    for cuts in range(1 << len(edges)):
        at = [0] + [b + 1 for b in range(len(edges)) if cuts >> b & 1] + [n]
        total = 0
        for a, e in zip(at, at[1:]):
            low = min(edges[a:e - 1], default=0)
            total += (e - a - 1) * (low if low >= least else 0)
        best = max(best, total)
    return best


@pytest.mark.parametrize("seed", range(60))
def test_the_cut_that_saves_the_most(seed):
    rng = np.random.default_rng(seed)
    edges = [int(x) for x in rng.choice([0, 1, 2, 3, 5, 9, 40], rng.integers(1, 10))]
    if seed % 3 == 0:  # stretches of equal neighbours
        edges = [e for e in edges[:4] for _ in range(int(rng.integers(1, 4)))]
    for least in (1, 3):
        tables = tables_of(edges)
        off, shared = groups_of(tables, least)
        assert off[0] == 0 and off[-1] == len(tables) and np.all(np.diff(off) > 0)
        for a, e, n in zip(off, off[1:], shared):
            assert n == 0 or n >= least
            assert n == 0 or e - a > 1
            assert all(t[:n] == tables[a][:n] for t in tables[a:e])
        assert saved(off, shared) == most(edges, least)


def doc(pages, n, head):
    body = list(range(1000, 1000 + pages))
    return [head + body + [10 ** 5 + i] for i in range(n)]


@pytest.mark.parametrize("order", ["before", "behind", "both", "between"])
def test_a_weakly_related_sequence_keeps_no_group_from_sharing(order):
    """64 questions about one document behind a page of instructions, and sequences
    that share that page alone."""
    from test_cpu_long_plan import Host
    group = doc(1000, 64, [7])
    loose = [[7] + list(range(5000 + 100 * i, 5080 + 100 * i)) for i in range(2)]
    tables = {"before": loose[:1] + group, "behind": group + loose[:1],
              "both": loose[:1] + group + loose[1:],
              "between": group[:32] + loose + group[32:]}[order]
    off, shared = groups_of(tables)
    assert sorted(shared)[-1] == 1001
    members = sum(e - a for a, e, n in zip(off, off[1:], shared) if n == 1001)
    assert members == 64
    kv = np.cumsum([0] + [len(t) for t in tables])
    pages = np.concatenate(tables)
    remap = {p: i for i, p in enumerate(sorted(set(pages.tolist())))}
    pages = np.array([remap[p] for p in pages.tolist()])
    host = Host(64, 8, 128, 16, len(tables), 1100, len(remap))
    host.prepare(np.arange(len(tables) + 1), kv, pages, [3] * len(tables))
    info = _lib.LongPlanInfo()
    assert host.lib.fe_long_plan_get_info(host.h, ctypes.byref(info)) == 0
    halves = 2 if order == "between" else 1
    assert info.shared_groups == halves
    assert info.shared_tiles >= (64 - halves) * 1000 * 8


def test_documents_of_their_own_each_share():
    tables = sum((doc(50 + i, 3 + i, [7])[:] for i in range(4)), [])
    # the documents differ behind the instruction page
    for i, (a, e) in enumerate(((0, 3), (3, 7), (7, 12), (12, 18))):
        for t in tables[a:e]:
            t[1:-1] = [p + 10000 * i for p in t[1:-1]]
    assert groups_of(tables) == ([0, 3, 7, 12, 18], [51, 52, 53, 54])


def test_one_page_for_all_is_one_group():
    assert groups_of(tables_of([1] * 30)) == ([0, 31], [1])
    assert groups_of(tables_of([4] * 1500)) == ([0, 1501], [4])


def test_a_large_batch_of_different_neighbours():
    rng = np.random.default_rng(5)
    edges = [int(x) for x in rng.integers(0, 60, 1023)]
    off, shared = groups_of(tables_of(edges))
    assert saved(off, shared) >= sum(edges[::2])  # pairs of neighbours, or better
