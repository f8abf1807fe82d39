"""The planners of shared-prefix and scored plans without a GPU: every query
row sees each of its keys exactly once through the lists; refusals."""
import ctypes

import numpy as np
import pytest

import fekv
from fekv import _lib
from fekv.ops import GROUP_DTYPE, ITEM_DTYPE, SEQ_DTYPE, FeError, check

ROW = np.dtype([(n, "<i4") for n in ("own_unit", "own_blocks", "own_rows", "own_p", "pre_unit",
                                     "pre_blocks", "pre_rows", "pre_p")])
UNIT = np.dtype([(n, "<i4") for n in ("part0", "n", "rec_floats", "rows")])
KEY = np.dtype([(n, "<i4") for n in ("q_row0", "qrows", "length", "page_off", "kvh", "key_mode",
                                     "kt0", "kt1", "part", "group", "seq", "pad")])
CHUNK = np.dtype([(n, "<i4") for n in ("block0", "blocks", "length", "page_off", "fresh", "t0")])


class Host:
    def __init__(self, hq, hkv, dim, page, batch, pages, blocks, scored=False, max_keys=0,
                 ctas=148):
        self.lib = _lib.load()
        self.h = ctypes.c_void_p()
        self.hq, self.hkv, self.dim, self.page, self.scored = hq, hkv, dim, page, scored
        self.item = 256 if dim == 128 else 128  # packed rows of a row item
        check(self.lib.fe_long_plan_create_host(hq, hkv, dim, page, batch, pages, 1, blocks,
                                                int(scored), max_keys, ctas, ctypes.byref(self.h)),
              "create")

    def __del__(self):
        self.lib.fe_long_plan_destroy(self.h)

    def prepare(self, qo, kv, pages, last, groups=None, fresh=None, graph=0, batch=None, rows=None):
        qo, kv, pages, last = (np.asarray(x, np.int32) for x in (qo, kv, pages, last))
        batch = len(kv) - 1 if batch is None else batch
        rows = int(qo[-1]) if rows is None else rows
        a = [x.ctypes.data for x in (qo, kv, pages, last)]
        if self.scored:
            f = None if fresh is None else np.asarray(fresh, np.int32)
            check(self.lib.fe_scored_plan_prepare(self.h, *a, None if f is None else f.ctypes.data,
                                                  batch, rows, graph, None), "prepare")
        else:
            off, shared = fekv.shared_prefixes(kv, pages) if groups is None else groups
            off, shared = np.asarray(off, np.int32), np.asarray(shared, np.int32)
            check(self.lib.fe_shared_plan_prepare(self.h, *a, off.ctypes.data, shared.ctypes.data,
                                                  len(shared), batch, rows, graph, None), "prepare")
        n = ctypes.c_int64(0)
        check(self.lib.fe_long_plan_debug_meta(self.h, None, 0, ctypes.byref(n)), "meta")
        buf = np.zeros(n.value, np.uint8)
        check(self.lib.fe_long_plan_debug_meta(self.h, buf.ctypes.data, n.value, ctypes.byref(n)),
              "meta")
        return Meta(buf)


class Meta:
    def __init__(self, buf):
        h = buf[:128].view(np.int32)
        take = lambda off, n, dt: buf[off:off + n * np.dtype(dt).itemsize].view(dt)  # noqa: E731
        self.lists = []
        for c in range(3):
            n, g, grid = int(h[c]), int(h[3 + c]), int(h[6 + c])
            self.lists.append((take(h[9 + c], grid + 1, "<i4") if grid else np.zeros(1, int),
                               take(h[12 + c], n, ITEM_DTYPE), take(h[15 + c], g, GROUP_DTYPE)))
        self.batch, self.rows, self.H = (int(h[i]) for i in (18, 19, 24))
        sink, info, chunk, u0, u1, n_chunks, key = (int(x) for x in h[25:32])
        seqs = int(h[20])
        self.info = take(info, self.rows, ROW)
        self.units = [take(u0, (u1 - u0) // UNIT.itemsize, UNIT),
                      take(u1, ((key or seqs) - u1) // UNIT.itemsize, UNIT)]
        self.seqs = take(seqs, (info - seqs) // SEQ_DTYPE.itemsize, SEQ_DTYPE)
        if key:  # the key kernel's items say the same
            k = take(key, int(h[2]), KEY)
            w = self.lists[2][1]
            for n in ("kvh", "key_mode", "kt0", "kt1", "part", "group", "seq"):
                np.testing.assert_array_equal(k[n], w[n])
            for n, of in (("q_row0", "q_row0"), ("qrows", "qrows"), ("length", "length"),
                          ("page_off", "page_off")):
                np.testing.assert_array_equal(k[n], self.seqs[w["seq"]][of])
        self.chunks = take(chunk, n_chunks, CHUNK)
        self.sink = buf[sink:int(h[21])].view("<i8")
        self.pages = buf[int(h[21]):].view("<i4")


def coverage(m, host, view):
    """Per query row and KV head: the pages' slots that its records cover, by
    the tables that the kernels read."""
    G, H, page = host.hq // host.hkv, m.H, host.page
    pieces = {}
    for c in (view, 2):
        off, items, groups = m.lists[c]
        assert off[0] == 0 and off[-1] == len(items) and (np.diff(off) >= 0).all()
        for it in items:
            pieces.setdefault((c, int(it["group"])), []).append(it)
        for (cc, g), its in pieces.items():
            if cc == c and g >= 0:
                n = groups[g]["nsplit"]
                assert len(its) == n
                assert sorted(i["part"] for i in its) == [groups[g]["part0"] + s *
                                                          groups[g]["rec_floats"] for s in range(n)]
    spans = []  # records do not overlap
    for c in (view, 2):
        for g in m.lists[c][2]:
            spans.append((g["part0"], g["part0"] + g["nsplit"] * g["rec_floats"]))
    spans.sort()
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))

    first = {}  # records' pieces by where they begin
    for c in (view, 2):
        for g, x in enumerate(m.lists[c][2]):
            first[int(x["part0"])] = (c, g)

    def keys(unit, blocks, p, P, kvh, qrow, causal):
        u = m.units[view][unit + (kvh * blocks + p // host.item if blocks else kvh // H)]
        if u["n"] == 0:
            return None
        c, g = first[int(u["part0"])]
        x = m.lists[c][2][g]
        assert (u["n"], u["rec_floats"], u["rows"]) == (x["nsplit"], x["rec_floats"], x["rows"])
        row = p % host.item if blocks else kvh % H * P + p
        assert row + G <= u["rows"] and u["rows"] * (host.dim + 2) <= u["rec_floats"]
        out = []
        for it in pieces[(c, g)]:
            s = m.seqs[it["seq"]]
            assert it["kvh"] <= kvh < it["kvh"] + (1 if blocks else H)
            if blocks:
                assert it["rb0"] * 16 == p // host.item * host.item
            i = qrow - s["q_row0"]
            assert 0 <= i < s["qrows"] and P == s["qrows"] * G
            hides = causal and it["key_mode"] != 2
            limit = s["length"] - s["qrows"] + i + 1 if hides else s["length"]
            t = np.arange(it["kt0"] * 16, min(it["kt1"] * 16, limit))
            out.append(m.pages[s["page_off"] + t // page].astype(np.int64) * page + t % page)
        return np.concatenate(out)

    direct = {}
    for c in (view, 2):
        for it in m.lists[c][1]:
            if it["group"] < 0:
                direct.setdefault((c, int(it["seq"])), []).append(it)
    seen = []
    for r in range(m.rows):
        x = m.info[r]
        for kvh in range(host.hkv):
            own = keys(x["own_unit"], x["own_blocks"], x["own_p"], x["own_rows"], kvh, r, view == 1)
            if own is None:
                seen.append(None)
                continue
            pre = keys(x["pre_unit"], x["pre_blocks"], x["pre_p"], x["pre_rows"], kvh, r,
                       view == 1) if x["pre_unit"] >= 0 else np.zeros(0, int)
            seen.append(np.sort(np.concatenate([own, pre])))
    return seen, direct


def step(groups, page, seed=0):
    """(qo, kv, pages, last), tables, lens, rows of groups (prefix pages,
    [(own tokens, rows)])."""
    rng = np.random.default_rng(seed)
    need = sum(p + sum(-(-n // page) for n, _ in m) for p, m in groups)
    order = list(rng.permutation(need + 3))
    tables, lens, rows = [], [], []
    for p, members in groups:
        head = [order.pop() for _ in range(p)]
        for n, r in members:
            tables.append(head + [order.pop() for _ in range(-(-n // page))])
            lens.append(p * page + n)
            rows.append(r)
    cum = lambda v: np.cumsum([0] + list(v))  # noqa: E731
    return (cum(rows), cum(map(len, tables)), np.concatenate(tables),
            [(n - 1) % page + 1 for n in lens]), tables, lens, rows, need + 3


LAYOUTS = [
    [(32, [(1, 1), (5, 1), (33, 1)]), (0, [(70, 1)])],
    [(24, [(n, 1) for n in range(1, 61)])],
    [(20, [(7, 1)] * 40), (40, [(n, 1) for n in range(3, 40)]), (1, [(2, 1), (9, 1)])],
    [(30, [(4, 4)] * 9 + [(20, 3), (3, 0), (16, 16)] + [(5, 5)] * 8)],
    [(26, [(300, 300)] + [(n, 1) for n in range(1, 30)]), (2, [(40, 40)])],
    [(0, [(1, 1)])],
]


@pytest.mark.parametrize("graph", [0, 1])
@pytest.mark.parametrize("shape", [(16, 8, 128, 16), (32, 4, 128, 32), (6, 3, 128, 48),
                                   (16, 2, 256, 16), (16, 1, 128, 16)])
@pytest.mark.parametrize("layout", range(len(LAYOUTS)))
def test_every_key_once(layout, shape, graph):
    hq, hkv, dim, page = shape
    meta, tables, lens, rows, blocks = step(LAYOUTS[layout], page, layout)
    host = Host(hq, hkv, dim, page, len(tables), max(map(len, tables)), blocks)
    m = host.prepare(*meta, graph=graph)
    for view in (0, 1):
        seen, direct = coverage(m, host, view)
        at = 0
        for b, (t, n, r) in enumerate(zip(tables, lens, rows)):
            for i in range(r):
                limit = n - r + i + 1 if view else n
                k = np.arange(limit)
                want = np.sort(np.asarray(t)[k // page] * page + k % page)
                for kvh in range(hkv):
                    got = seen[(at + i) * hkv + kvh]
                    if got is not None:
                        np.testing.assert_array_equal(got, want)
            if r and any(seen[at * hkv + kvh] is None for kvh in range(hkv)):
                # a unit that writes its output itself holds the whole key range
                its = direct.get((view, b), []) + direct.get((2, b), [])
                assert its and all(it["kt0"] == 0 for it in its)
                assert max(it["kt1"] for it in its) == -(-n // 16)
            at += r


@pytest.mark.parametrize("shape", [(16, 8, 128, 16), (12, 4, 128, 16), (6, 3, 128, 48),
                                   (16, 2, 256, 16), (16, 1, 128, 16)])
def test_scored_blocks_cover_rows_and_keys(shape):
    hq, hkv, dim, page = shape
    members = [(1, 1), (900, 32), (33, 33), (37, 0), (20, 3)]
    meta, tables, lens, rows, blocks = step([(0, members)], page)
    cap = sum(r * (n + 15) for n, r in zip(lens, rows))
    host = Host(hq, hkv, dim, page, len(tables), max(map(len, tables)), blocks, True, cap)
    fresh = [1, 900, 5, 0, 20]
    m = host.prepare(*meta, fresh=fresh)
    seen, _ = coverage(m, host, 1)
    at = 0
    spans = []
    for b, (t, n, r) in enumerate(zip(tables, lens, rows)):
        for i in range(r):
            k = np.arange(n - r + i + 1)
            want = np.sort(np.asarray(t)[k // page] * page + k % page)
            for kvh in range(hkv):
                np.testing.assert_array_equal(seen[(at + i) * hkv + kvh], want)
        at += r
        if r:
            mine = [c for c in m.chunks if c["page_off"] == meta[1][b]]
            assert [c["t0"] for c in mine] == list(range(0, n, 512))
            assert all(c["length"] == n and c["fresh"] == n - fresh[b] for c in mine)
            units = [m.info[int(m.seqs[mine[0]["block0"] + j]["q_row0"])]["own_unit"]
                     for j in range(mine[0]["blocks"])]  # of its row blocks
            assert np.array_equal(np.diff(units), [hkv // m.H] * (len(units) - 1))
            s = m.seqs[mine[0]["block0"]:mine[0]["block0"] + mine[0]["blocks"]]
            assert s["qrows"].sum() == r and (s["qrows"] * (hq // hkv) <= 16).all()
            assert s["length"][-1] == n
            spans += list(s)
    # raw scores lie one behind the other, within what the plan holds
    G = hq // hkv
    sink = [0]
    for s in spans:
        P = s["qrows"] * G
        sink.append(sink[-1] + hkv * -(-s["length"] // 16) * 16 * (P + P % 2))
    np.testing.assert_array_equal(m.sink[:len(spans)], sink[:-1])
    assert sink[-1] <= cap * hkv * (G + G % 2)


def refused(status, call, text=None):
    with pytest.raises(FeError, match=text) as e:
        call()
    assert e.value.status == status


def test_refusals():
    meta, tables, lens, rows, blocks = step([(8, [(5, 1)] * 4)], 16)
    qo, kv, pages, last = meta
    host = Host(16, 8, 128, 16, 4, 16, blocks)
    bad = _lib.FE_ERR_INVALID_ARGUMENT
    for groups in (([0, 3], [8]), ([1, 4], [8]), ([0, 3, 2, 4], [8, 8, 8]), ([0, 4], [-1]),
                   ([0, 4], [9]), ([0, 4], [10])):
        refused(bad, lambda: host.prepare(*meta, groups=groups))
    other = pages.copy()
    other[kv[2] + 3] = other[kv[1] - 1]
    refused(bad, lambda: host.prepare(qo, kv, other, last, groups=([0, 4], [8])), "does not begin")
    refused(bad, lambda: host.prepare(qo, kv, pages, [17, 1, 1, 1]))
    refused(bad, lambda: host.prepare(qo, kv, np.where(pages == pages[0], blocks + 1, pages), last))
    refused(_lib.FE_ERR_CAPACITY, lambda: Host(16, 8, 128, 16, 3, 2, blocks).prepare(*meta))
    refused(_lib.FE_ERR_CONTEXT, lambda: host.prepare([0, 200, 201, 202, 203], kv, pages, last))
    host.prepare(*meta, graph=1)
    refused(bad, lambda: host.prepare([0, 1, 2, 3, 5], kv, pages, [5, 5, 5, 5], graph=1), "graph")
    s = Host(16, 8, 128, 16, 4, 16, blocks, True, 4 * 144)
    refused(bad, lambda: s.prepare(*meta), "twice")
    meta, tables, lens, rows, blocks = step([(0, [(133, 1)] * 4)], 16)
    s = Host(16, 8, 128, 16, 4, 16, blocks, True, 4 * 144)
    s.prepare(*meta)
    for fresh in ([-1, 1, 1, 1], [1, 1, 1, 134]):
        refused(bad, lambda: s.prepare(*meta, fresh=fresh), "fresh")
    refused(_lib.FE_ERR_CAPACITY,
            lambda: Host(16, 8, 128, 16, 4, 16, blocks, True, 4 * 144 - 1).prepare(*meta),
            "max_keys")
    for wrong in ((16, 8, 64, 16), (16, 5, 128, 16), (34, 2, 128, 16), (16, 8, 128, 24)):
        refused(_lib.FE_ERR_UNSUPPORTED, lambda: Host(*wrong, 4, 16, blocks))
    lib = _lib.load()
    p = ctypes.c_void_p()
    assert lib.fe_long_plan_create_host(16, 8, 128, 16, 4, 16, 7, 9, 0, 0, 1,
                                        ctypes.byref(p)) == bad
    assert lib.fe_shared_attn_run(None, 1, 1, 1, 1, 1, None) == bad
    assert lib.fe_shared_attn_run(host.h, 16, 16, 16, 16, 1, None) == bad  # host-only
    assert lib.fe_scored_attn_run(s.h, 16, 16, 16, 16, 16, None) == bad
    assert lib.fe_scored_plan_prepare(host.h, None, None, None, None, None, 0, 0, 0, None) == bad
    assert lib.fe_shared_plan_prepare(s.h, None, None, None, None, None, None, 0, 0, 0, 0,
                                      None) == bad


def test_an_empty_step():
    host = Host(16, 8, 128, 16, 4, 16, 20)
    m = host.prepare([0], [0], np.zeros(0, np.int32), np.zeros(0, np.int32))
    assert m.rows == 0 and not len(m.lists[2][1])
    s = Host(16, 8, 128, 16, 4, 16, 20, True, 0)
    assert s.prepare([0], [0], np.zeros(0, np.int32), np.zeros(0, np.int32)).rows == 0


def test_groups_are_found():
    def groups(*tables, least=1):
        kv = np.cumsum([0] + [len(t) for t in tables])
        off, shared = fekv.shared_prefixes(kv, np.concatenate(tables), least)
        return off.tolist(), shared.tolist()

    a, b = list(range(10)), list(range(50, 60))
    assert groups(a + [11], a + [12], b + [13], b + [14, 15]) == ([0, 2, 4], [10, 10])
    assert groups(a, a, a) == ([0, 3], [10])
    assert groups(a, b, a) == ([0, 1, 2, 3], [0, 0, 0])
    # a neighbour that shares less than half begins anew; one that shares more lowers it
    assert groups(a + [11], a + [12], a[:7] + [13], a[:2] + [14]) == ([0, 3, 4], [7, 0])
    assert groups(a + [11], a[:3] + [12], least=4) == ([0, 1, 2], [0, 0])
    off, shared = fekv.shared_prefixes([0], [])
    assert off.tolist() == [0] and not len(shared)
    with pytest.raises(ValueError):
        fekv.shared_prefixes([0, 3], [1, 2])
    with pytest.raises(FeError):
        fekv.shared_prefixes([0, 2], [1, 2], 0)
