"""Scored plans serve every step within max_keys: prompts of one sequence, many
query rows, many heads. Host planner only, needs no GPU."""
import numpy as np
import pytest

from fekv import _lib
from fekv.ops import FeError
from test_cpu_long_plan import Host, coverage


def prompts(lens, rows, page=16):
    cum = lambda v: np.cumsum([0] + list(v))  # noqa: E731
    pages = [-(-n // page) for n in lens]
    return cum(rows), cum(pages), np.arange(sum(pages)), [(n - 1) % page + 1 for n in lens]


def keys(lens, rows):
    return sum(r * (-(-n // 16) * 16) for n, r in zip(lens, rows))


# (heads, head_dim, max_batch, keys and query rows of each sequence)
STEPS = [((32, 8, 128), 1, [4000], [4000]), ((128, 8, 128), 1, [1024], [1024]),
         ((32, 8, 128), 4, [2048] * 4, [2048] * 4), ((32, 8, 128), 4, [8192, 1, 1, 1], [8192, 1, 1, 1]),
         ((16, 1, 128), 1, [9000], [9000]), ((16, 16, 128), 1, [3001], [3001]),
         ((40, 8, 128), 2, [50, 4099], [50, 4099]), ((32, 2, 256), 1, [8300], [8300]),
         ((5, 5, 256), 1, [6000], [6000]), ((128, 8, 128), 64, [32] * 64, [32] * 64),
         ((8, 8, 128), 300, [17] * 300, [17] * 300), ((64, 4, 128), 512, [16] * 512, [1] * 512)]


@pytest.mark.parametrize("graph", [0, 1])
@pytest.mark.parametrize("n", range(len(STEPS)))
def test_steps_within_max_keys(n, graph):
    (hq, hkv, dim), batch, lens, rows = STEPS[n]
    pages = [-(-x // 16) for x in lens]
    host = Host(hq, hkv, dim, 16, batch, max(pages), sum(pages), True, keys(lens, rows))
    m = host.prepare(*prompts(lens, rows), graph=graph)
    assert m.rows == sum(rows)
    G, per = hq // hkv, 16 // (hq // hkv)
    blocks = sum(-(-r // per) for r in rows)
    assert len(m.units[1]) == blocks * (hkv // m.H) and (m.units[1]["n"] > 0).all()
    assert (m.info["own_unit"] >= 0).all()
    off, items, groups = m.lists[2]
    assert len(items) >= len(groups) == len(m.units[1]) and off[-1] == len(items)
    # the records lie one behind the other, offsets within 31 bits
    end = groups["part0"].astype(np.int64) + groups["nsplit"].astype(np.int64) * groups["rec_floats"]
    np.testing.assert_array_equal(groups["part0"][1:], end[:-1])
    assert groups["part0"][0] == 0 and end[-1] < 2 ** 31
    with pytest.raises(FeError, match="max_keys") as e:
        Host(hq, hkv, dim, 16, batch, max(pages), sum(pages), True,
             keys(lens, rows) // 16 // 16).prepare(*prompts(lens, rows), graph=graph)
    assert e.value.status == _lib.FE_ERR_CAPACITY


def test_every_key_once_in_a_long_prompt():
    """More row blocks than the plan's batch and heads used to allow (64 each)."""
    lens = rows = [1040]
    host = Host(128, 8, 128, 16, 1, 65, 65, True, keys(lens, rows))
    meta = prompts(lens, rows)
    m = host.prepare(*meta)
    assert len(m.lists[2][1]) > 8192
    seen, _ = coverage(m, host, 1)
    for i in range(rows[0]):
        want = np.arange(i + 1)
        for h in range(8):
            np.testing.assert_array_equal(seen[i * 8 + h], want)


def test_records_beyond_31_bits_are_refused():
    lens = rows = [16] * 8192
    host = Host(128, 8, 128, 16, 8192, 1, 8192, True, keys(lens, rows))
    with pytest.raises(FeError, match="workspace") as e:
        host.prepare(*prompts(lens, rows))
    assert e.value.status == _lib.FE_ERR_CAPACITY
