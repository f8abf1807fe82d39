"""The 8-bit KV cache without a GPU: the restatement's own e4m3 against
torch's, the C ABI's refusals, and the planner's lists for an 8-bit plan."""
import ctypes

import numpy as np
import pytest

import fekv
import kv8_ref as ref
from fekv import _lib

P = ctypes.c_void_p(4096)
ODD = ctypes.c_void_p(4098)


def test_e4m3_restatement_agrees_with_torch():
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal(5000) * np.exp2(rng.integers(-14, 9, 5000)),
                        ref.decode_e4m3(np.arange(256, dtype=np.uint8)),
                        [0.0, -0.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -11, 17.0, 19.0]])
    x = np.clip(x, -448, 448).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    got = ref.encode_e4m3(x.astype(np.float64))
    nan = np.isnan(x)
    assert np.array_equal(got[~nan], want[~nan])
    back = torch.from_numpy(want).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(ref.decode_e4m3(want), back, equal_nan=True)


@pytest.mark.parametrize("amax,e", [(448.0, 0), (448.1, 1), (224.0, -1), (1.75, -8), (1.76, -7),
                                    (0.0, -32), (1e-30, -32), (1e38, 64)])
def test_scale_of_a_magnitude(amax, e):
    assert ref.needed(amax) == e


def append_args(**kw):
    a = dict(q=P, q_out=P, k=P, v=P, kc=P, vc=P, ke=P, ve=P, slots=P, pos=P, cache=P, rows=1, hq=8,
             hkv=4, dim=128, rot=128, most=10, dtype=1, cs=32, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=2), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(rows=-1), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(hkv=0), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(hq=-1), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(cs=0), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(cs=24), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(dim=64), _lib.FE_ERR_UNSUPPORTED),
    (dict(rot=136), _lib.FE_ERR_UNSUPPORTED),
    (dict(rot=4), _lib.FE_ERR_UNSUPPORTED),
    (dict(rot=-8), _lib.FE_ERR_UNSUPPORTED),
    (dict(most=0), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(k=None), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(q_out=None), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(ve=None), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(pos=None), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(cache=None), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(k=ODD), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(vc=ODD), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(rows=0), _lib.FE_OK),
])
def test_append_refusals(kw, status):
    assert fekv.load().fe_kv8_append(*append_args(**kw)) == status


def gather_args(**kw):
    a = dict(codes=P, exps=P, out=P, kv=P, pages=P, last=P, off=P, batch=1, max_len=4, page=16,
             hkv=2, dim=128, dtype=0, cs=32, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=5), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(batch=-1), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(page=24), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(dim=24), _lib.FE_ERR_UNSUPPORTED),
    (dict(batch=65536), _lib.FE_ERR_CAPACITY),
    (dict(out=None), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(codes=ODD), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(batch=0), _lib.FE_OK),
    (dict(max_len=0), _lib.FE_OK),
])
def test_gather_refusals(kw, status):
    assert fekv.load().fe_kv8_gather(*gather_args(**kw)) == status


def copy_args(**kw):
    one = (ctypes.c_void_p * 1)(4096)
    a = dict(kc=one, vc=one, ke=one, ve=one, layers=1, src=P, dst=P, ntok=P, copies=1, page=16,
             hkv=2, dim=128, pages=4, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,status", [
    (dict(layers=-1), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(layers=_lib.FE_MAX_LAYERS + 1), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(page=8), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(pages=0), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(copies=65536), _lib.FE_ERR_CAPACITY),
    (dict(src=None), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(ve=(ctypes.c_void_p * 1)(None)), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(kc=(ctypes.c_void_p * 1)(4100)), _lib.FE_ERR_INVALID_ARGUMENT),
    (dict(copies=0), _lib.FE_OK),
    (dict(layers=0), _lib.FE_OK),
])
def test_copy_refusals(kw, status):
    assert fekv.load().fe_kv8_copy_blocks(*copy_args(**kw)) == status


def test_attention_refusals():
    lib = fekv.load()
    run = lib.fe_kv8_attn_run
    assert run(None, P, P, P, P, P, P, 1, None) == _lib.FE_ERR_INVALID_ARGUMENT
    plan = fekv.HostKv8Plan(8, 4, 128, 16, 4, 8, True, 64)
    assert run(plan.handle, P, P, P, P, P, P, 1, None) == _lib.FE_ERR_INVALID_ARGUMENT
    out = ctypes.c_void_p()
    for bad, status in [((8, 4, 64), _lib.FE_ERR_UNSUPPORTED), ((8, 3, 128), _lib.FE_ERR_UNSUPPORTED),
                        ((34, 2, 128), _lib.FE_ERR_UNSUPPORTED)]:
        assert lib.fe_kv8_plan_create_host(*bad, 16, 4, 8, 1, 64, 10,
                                           ctypes.byref(out)) == status
    with pytest.raises(fekv.FeError):  # fewer keys than rows
        plan.prepare([0, 5], [0, 1], [3], [4])


def test_row_lists_are_cut_and_cover_every_key():
    """Every (sequence, KV head, 128-row group) has its keys covered once, in
    pieces at whole tiles, and the pieces' records do not overlap."""
    plan = fekv.HostKv8Plan(16, 4, 128, 16, 4, 600, True, 2000, grid_cap=296)
    lens, rows = [9000, 40, 700], [20, 40, 1]
    need = [-(-n // 16) for n in lens]
    kv = np.cumsum([0] + need)
    meta = plan.prepare(np.cumsum([0] + rows), kv, np.arange(kv[-1]),
                        [(n - 1) % 16 + 1 for n in lens])
    for view, causal in ((meta["views"][0], False), (meta["views"][1], True)):
        seen = {}
        spans = []
        for it in view["items"]:
            seen.setdefault((int(it["seq"]), int(it["kvh"]), int(it["rb0"])), []).append(
                (int(it["kt0"]), int(it["kt1"])))
            if it["part"] >= 0:
                n = view["groups"][it["group"]]["rec_floats"]
                spans.append((int(it["part"]), int(it["part"] + n)))
        for (seq, _, rb0), parts in seen.items():
            parts.sort()
            last = min(rows[seq] * 4, rb0 * 16 + 128) - 1
            keys = lens[seq] - rows[seq] + last // 4 + 1 if causal else lens[seq]
            assert parts[0][0] == 0 and parts[-1][1] == -(-keys // 16)
            assert all(a[1] == b[0] for a, b in zip(parts, parts[1:]))
        assert len(seen) == 4 * (1 + 2)
        spans.sort()
        assert spans and all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
    plan.close()
