"""Arguments that the calls for long shared prompts (rotary positions with
several axes, attention over shared prefixes and with scores, eviction) refuse
before anything is launched, beside those of test_cpu_long_plan.py. None needs
a GPU."""
import ctypes

import numpy as np
import pytest

import fekv
from fekv import _lib
from test_cpu_8bit_refusals import lib, placed  # noqa: F401  (lib is a fixture)

torch = pytest.importorskip("torch")

BAD, UNSUPPORTED, CAPACITY = (_lib.FE_ERR_INVALID_ARGUMENT, _lib.FE_ERR_UNSUPPORTED,
                              _lib.FE_ERR_CAPACITY)
P = 1 << 20  # an address that is never read: the call is refused first


# ---------------------------------------------------------------------------
# the C calls
# ---------------------------------------------------------------------------

def axes_c(**kw):
    a = dict(q=P, k=P, v=P, k_out=None, kc=P, vc=P, slots=P, pos=P, axes=3,
             pairs=bytes([0, 1, 2, 0]), cache=P, rows=2, hq=2, hkv=1, dim=16, rot=8, most=10,
             dtype=0, cs=32, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return fekv.load().fe_rope_axes_append(*a.values())


@pytest.mark.parametrize("kw,status", [
    (dict(axes=0), UNSUPPORTED), (dict(axes=5), UNSUPPORTED), (dict(axes=2), BAD),
    (dict(dim=18), UNSUPPORTED), (dict(rot=6), UNSUPPORTED), (dict(rot=20), UNSUPPORTED),
    (dict(rot=516, dim=520, pairs=bytes(258)), UNSUPPORTED), (dict(dtype=7), BAD),
    (dict(rows=-1), BAD), (dict(hq=-1), BAD), (dict(hkv=0), BAD), (dict(most=0), BAD),
    (dict(pairs=None), BAD), (dict(k=None), BAD), (dict(q=None), BAD), (dict(v=None), BAD),
    (dict(kc=None), BAD), (dict(vc=None), BAD), (dict(slots=None), BAD), (dict(pos=None), BAD),
    (dict(cache=None), BAD), (dict(cs=0), BAD), (dict(k=P + 2), BAD), (dict(cache=P + 2), BAD),
    (dict(pos=P + 4), BAD), (dict(slots=P + 4), BAD), (dict(rows=(1 << 30) + 1), CAPACITY),
    (dict(hq=1 << 21), CAPACITY), (dict(hq=(1 << 31) - 1, hkv=(1 << 31) - 1), CAPACITY)])
def test_rope_axes_append(kw, status):
    assert axes_c(**kw) == status
    assert b"fe_rope_axes_append" in fekv.load().fe_last_error()


def test_no_rows_is_no_call():
    assert axes_c(rows=0, q=None, k=None) == _lib.FE_OK


def select_c(**kw):
    a = dict(scores=P, kv=P, pages=P, num_pages=3, last=P, kept=P, batch=1, max_len=40, hkv=2,
             page=16, budget=8, sink=1, recent=2, cs=64, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return fekv.load().fe_kv_select(*a.values())


@pytest.mark.parametrize("kw,status", [
    (dict(batch=-1), BAD), (dict(hkv=0), BAD), (dict(budget=-1), BAD), (dict(num_pages=-1), BAD),
    (dict(page=0), UNSUPPORTED), (dict(page=24), UNSUPPORTED), (dict(cs=0), BAD),
    (dict(cs=40), BAD), (dict(cs=1 << 31), BAD), (dict(sink=-1), BAD), (dict(recent=-1), BAD),
    (dict(sink=4, recent=5), BAD), (dict(sink=(1 << 31) - 1, recent=(1 << 31) - 1), BAD),
    (dict(max_len=-1), BAD), (dict(scores=None), BAD), (dict(kept=None), BAD),
    (dict(kv=None), BAD), (dict(pages=None), BAD), (dict(last=None), BAD),
    (dict(scores=P + 4), BAD), (dict(batch=1 << 20, hkv=1 << 12), CAPACITY)])
def test_select(kw, status):
    assert select_c(**kw) == status
    assert b"fe_kv_select" in fekv.load().fe_last_error()


def compact_c(**kw):
    a = dict(k=P, v=P, scores=P, kept=P, kv=P, pages=P, num_pages=3, last=P, dst_kv=None,
             dst_pages=None, num_dst=0, batch=1, hkv=2, dim=128, page=16, budget=8, dtype=0,
             cs=64, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return fekv.load().fe_kv_compact(*a.values())


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=9), BAD), (dict(dim=0), UNSUPPORTED), (dict(dim=12), UNSUPPORTED),
    (dict(dim=520), UNSUPPORTED), (dict(page=8), UNSUPPORTED), (dict(cs=63), BAD),
    (dict(k=None), BAD), (dict(v=None), BAD), (dict(kept=None), BAD), (dict(last=None), BAD),
    (dict(k=P + 8), BAD), (dict(v=P + 8), BAD), (dict(dst_kv=P), BAD), (dict(dst_pages=P), BAD),
    (dict(dst_kv=P, dst_pages=P, num_dst=-1), BAD), (dict(batch=-1), BAD)])
def test_compact(kw, status):
    assert compact_c(**kw) == status
    assert b"fe_kv_compact" in fekv.load().fe_last_error()


def test_nothing_to_select_or_move_is_no_call():
    for call in (select_c, compact_c):
        assert call(batch=0, kv=None, pages=None, last=None) == _lib.FE_OK
    assert select_c(budget=0, sink=0, recent=0, kept=None) == _lib.FE_OK
    assert compact_c(budget=0, kept=None) == _lib.FE_OK


@pytest.mark.parametrize("scored", [False, True])
@pytest.mark.parametrize("kw,status", [
    (dict(dim=64), UNSUPPORTED), (dict(hq=5), UNSUPPORTED), (dict(hq=34), UNSUPPORTED),
    (dict(page=24), UNSUPPORTED), (dict(batch=0), BAD), (dict(pages=0), BAD),
    (dict(dtype=5), BAD), (dict(blocks=0), BAD), (dict(blocks=(1 << 31) - 1), BAD),
    (dict(batch=1 << 20, pages=1 << 12), CAPACITY)])
def test_plans(kw, status, scored):
    a = dict(hq=8, hkv=2, dim=128, page=16, batch=2, pages=4, dtype=0, blocks=8)
    a.update(kw)
    h = ctypes.c_void_p()
    L = fekv.load()
    rc = (L.fe_scored_plan_create(*a.values(), 1024, ctypes.byref(h)) if scored else
          L.fe_shared_plan_create(*a.values(), ctypes.byref(h)))
    assert rc == status and not h.value


# ---------------------------------------------------------------------------
# the Python calls: shapes, types, layouts, devices
# ---------------------------------------------------------------------------

def t(*shape, dtype=torch.bfloat16, where=0):
    return placed(torch.zeros(*shape, dtype=dtype), where)


def i32(*v, where=0):
    return placed(torch.tensor(v, dtype=torch.int32), where)


def strided(x):
    return placed(torch.zeros(2 * x.shape[0], *x.shape[1:], dtype=x.dtype)[::2], 0)


def rope(axes=3, **kw):
    a = dict(q=t(5, 4, 128), k=t(5, 2, 128), pos=t(axes, 5, dtype=torch.int64),
             cache=t(9, 64, dtype=torch.float32), pairs=fekv.rope_sections((12, 10, 10)))
    a.update(kw)
    fekv.rope_axes(a["q"], a["k"], a["pos"], a["cache"], a["pairs"])


def append(**kw):
    a = dict(q=t(5, 4, 128), k=t(5, 2, 128), v=t(5, 2, 128), kc=t(32, 2, 128), vc=t(32, 2, 128),
             slots=t(5, dtype=torch.int64), pos=t(3, 5, dtype=torch.int64),
             cache=t(9, 64, dtype=torch.float32), pairs=fekv.rope_sections((12, 10, 10)),
             k_out=t(5, 2, 128))
    a.update(kw)
    fekv.rope_axes_append(a["q"], a["k"], a["v"], a["kc"], a["vc"], a["slots"], a["pos"],
                          a["cache"], a["pairs"], k_out=a["k_out"])


def select(**kw):
    a = dict(scores=t(2, 64, dtype=torch.float32), kv=i32(0, 2), pages=i32(0, 1), last=i32(5),
             kept=t(1, 2, 8, dtype=torch.int32))
    a.update(kw)
    fekv.select_tokens(a["scores"], a["kv"], a["pages"], a["last"], a["kept"], 16, 21)


def compact(**kw):
    a = dict(k=t(64, 2, 128), v=t(64, 2, 128), scores=t(2, 64, dtype=torch.float32),
             kept=t(1, 2, 8, dtype=torch.int32), kv=i32(0, 2), pages=i32(0, 1), last=i32(5),
             dst_kv=i32(0, 1), dst_pages=i32(2))
    a.update(kw)
    fekv.compact_tokens(a["k"], a["v"], a["scores"], a["kept"], a["kv"], a["pages"], a["last"],
                        16, a["dst_kv"], a["dst_pages"])


PYTHON = [
    (rope, dict(), None), (rope, dict(q=None), None), (rope, dict(q=t(5, 4, 64)), "q"),
    (rope, dict(q=t(4, 4, 128)), "q"), (rope, dict(q=t(5, 4, 128, dtype=torch.float16)), "q"),
    (rope, dict(q=t(5, 512)), "q"), (rope, dict(q=t(5, 4, 128, where=1)), "q"),
    (rope, dict(k=t(5, 2, 128, where=1)), "k"),
    (rope, dict(k=t(5, 2, 128, dtype=torch.float32), q=None), "float16 or bfloat16"),
    (rope, dict(k=strided(t(5, 2, 128))), "k"), (rope, dict(q=strided(t(5, 4, 128))), "q"),
    (rope, dict(pos=t(5, dtype=torch.int64)), "pos"),
    (rope, dict(pos=t(3, 4, dtype=torch.int64)), "pos"),
    (rope, dict(pos=t(3, 5, dtype=torch.int32)), "pos"), (rope, dict(pairs=bytes(31)), "pair_axis"),
    (rope, dict(pairs=[0] * 32), "pair_axis"),
    (rope, dict(cache=t(9, 64, dtype=torch.bfloat16)), "cache"), (append, dict(), None),
    (append, dict(k_out=None, q=None), None), (append, dict(v=t(5, 2, 64)), "v"),
    (append, dict(v=t(5, 2, 128, where=1)), "v"), (append, dict(k_out=t(4, 2, 128)), "k_out"),
    (append, dict(slots=t(4, dtype=torch.int64)), "slots"),
    (append, dict(slots=t(5, dtype=torch.int32)), "slots"), (append, dict(kc=t(31, 2, 128)), "kc"),
    (append, dict(vc=t(32, 2, 128, where=1)), "vc"),
    (append, dict(kc=strided(t(32, 2, 128))), "kc"),
    (append, dict(kc=t(32, 2, 128, dtype=torch.float16)), "kc"), (select, dict(), None),
    (select, dict(scores=t(64, dtype=torch.float32)), "scores"),
    (select, dict(scores=t(2, 64)), "scores"),
    (select, dict(scores=t(2, 64, dtype=torch.float32, where=1)), "scores"),
    (select, dict(kept=t(1, 2, 8, dtype=torch.int64)), "kept"),
    (select, dict(kept=t(1, 3, 8, dtype=torch.int32)), "kept"),
    (select, dict(kept=t(2, 8, dtype=torch.int32)), "kept"), (select, dict(kv=i32(0, 1, 2)), "kv"),
    (select, dict(last=i32(5, where=1)), "."), (select, dict(pages=t(2, dtype=torch.int64)), "."),
    (compact, dict(), None), (compact, dict(scores=None, dst_kv=None, dst_pages=None), None),
    (compact, dict(v=t(64, 2, 64)), "pools"),
    (compact, dict(v=t(64, 2, 128, dtype=torch.float16)), "v_pool"),
    (compact, dict(k=t(64, 2, 128, where=1)), "k_pool"),
    (compact, dict(scores=t(2, 48, dtype=torch.float32)), "scores"),
    (compact, dict(kept=t(1, 2, 8)), "kept"), (compact, dict(dst_kv=i32(0, 1, 1)), "dst_kv"),
    (compact, dict(dst_pages=None), "."), (compact, dict(dst_kv=None), "."),
    (compact, dict(dst_pages=i32(2, where=1)), "."),]


@pytest.mark.parametrize("n", range(len(PYTHON)))
def test_python_calls(lib, n):  # noqa: F811
    call, kw, word = PYTHON[n]
    if word is None:
        call(**kw)
        assert lib.count == 1
        return
    with pytest.raises((ValueError, TypeError), match=word):
        call(**kw)
    assert lib.count == 0


@pytest.mark.parametrize("sections,turns", [((), False), ((1, 2, 3, 4, 5), False), ((4, -1), False),
                                            ((2, 3), True), ((4, 4, 5), True)])
def test_sections(sections, turns):
    with pytest.raises(ValueError, match="sections"):
        fekv.rope_sections(sections, turns)


def test_sections_of_pairs():
    assert fekv.rope_sections((2, 1, 3)) == bytes([0, 0, 1, 2, 2, 2])
    assert fekv.rope_sections((4, 2, 1), True) == bytes([0, 1, 2, 0, 1, 0, 0])
    assert fekv.rope_sections((3, 3), True) == bytes([0, 1] * 3)


def plan(scored):
    if scored:
        return fekv.ScoredPlan(8, 2, 128, 16, 2, 4, True, 3, 4096)
    return fekv.SharedPlan(8, 2, 128, 16, 2, 4, True, 3)


def prepared(scored):
    p = plan(scored)
    p.prepare(np.array([0, 1, 3]), np.array([0, 2, 3]), np.array([0, 1, 2]), np.array([5, 16]),
              **({} if scored else {"groups": (np.array([0, 2]), np.array([0]))}))
    return p


@pytest.mark.parametrize("scored", [False, True])
@pytest.mark.parametrize("kw,word", [
    (dict(), None), (dict(q=t(2, 8, 128)), "q"), (dict(q=t(3, 4, 128)), "q"),
    (dict(q=t(3, 8, 128, dtype=torch.float16)), "q"), (dict(q=t(3, 8, 128, where=1)), "q"),
    (dict(out=t(2, 8, 128)), "out"), (dict(out=t(3, 8, 128, where=1)), "out"),
    (dict(k=t(48, 2, 128)), "pools"), (dict(v=t(80, 2, 128)), "pools"),
    (dict(k=t(64, 2, 128, where=1)), "k"), (dict(v=strided(t(64, 2, 128))), "v"),
    (dict(q=strided(t(3, 8, 128))), "q")])
def test_attention(lib, scored, kw, word):  # noqa: F811
    p = prepared(scored)
    a = dict(q=t(3, 8, 128), k=t(64, 2, 128), v=t(64, 2, 128), out=t(3, 8, 128))
    a.update(kw)
    extra = [t(2, 64, dtype=torch.float32)] if scored else []
    before = lib.count
    if word is None:
        p.attention(a["q"], a["k"], a["v"], *extra, a["out"])
        assert lib.count == before + 1
        return
    with pytest.raises(ValueError, match=word):
        p.attention(a["q"], a["k"], a["v"], *extra, a["out"])
    assert lib.count == before


@pytest.mark.parametrize("scores", [t(2, 48, dtype=torch.float32), t(3, 64, dtype=torch.float32),
                                    t(2, 64), t(2, 64, dtype=torch.float32, where=1)])
def test_attention_scores(lib, scores):  # noqa: F811
    p = prepared(True)
    before = lib.count
    with pytest.raises(ValueError, match="scores"):
        p.attention(t(3, 8, 128), t(64, 2, 128), t(64, 2, 128), scores, t(3, 8, 128))
    assert lib.count == before


@pytest.mark.parametrize("scored", [False, True])
def test_prepare(lib, scored, monkeypatch):  # noqa: F811
    p = plan(scored)
    ok = (np.array([0, 1, 3]), np.array([0, 2, 3]), np.array([0, 1, 2]), np.array([5, 16]))
    for i, short in ((0, ok[0][:2]), (2, ok[2][:2]), (3, ok[3][:1])):
        bad = list(ok)
        bad[i] = short
        with pytest.raises(ValueError):
            p.prepare(*bad)
    if scored:
        with pytest.raises(ValueError, match="fresh"):
            p.prepare(*ok, fresh=np.array([1]))
    else:
        with pytest.raises(ValueError, match="group_off"):
            p.prepare(*ok, groups=(np.array([0, 2]), np.array([0, 0])))
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1, raising=False)
    with pytest.raises(ValueError, match="cuda:0"):
        p.prepare(*ok)
