"""Forms of the 8-bit cache's operators that test_gpu_kv8.py does not reach,
against the same restatement in 64 bits (kv8_ref.py)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import fekv
import kv8_bounds as bounds
import kv8_ref as ref
from fekv import _lib
from test_gpu_kv8 import Step, codes_of, dev, exps_of, half, pool_of, random_pool

pytestmark = pytest.mark.gpu

DT = {True: torch.bfloat16, False: torch.float16}


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("byte", [0, 60, 94, 95, 191, 192, 255])
@pytest.mark.parametrize("hkv,dim,rows", [(8, 128, 1), (3, 256, 1), (8, 128, 1100), (8, 128, 4200)])
def test_append_reads_scales_outside_the_limits_as_every_reader_does(byte, hkv, dim, rows):
    """A scale byte outside the limits reads as the nearest within (attention
    and gather): an append that keeps tokens keeps those values, whichever way
    its own scale compares, and leaves a byte within the limits."""
    rng = np.random.default_rng(byte)
    lead = [(5, -14), (9, -40), (15, 60)]  # (tokens kept, exponent of the new ones)
    slots = [16 * (i + 1) + kept for i, (kept, _) in enumerate(lead)]
    slots += list(range(64, 64 + rows - 1))
    cs = (64 + rows + 31) // 16 * 16
    codes, exps = random_pool(rng, cs, hkv, dim)
    exps[:4] = byte
    k = half(rng.standard_normal((len(slots), hkv, dim)), True)
    for i, (_, e) in enumerate(lead):
        k[i] *= 2.0 ** e
    before = ref.values(codes, exps)
    kp, vp = pool_of(codes, exps), pool_of(codes, exps)
    kd = dev(k, torch.bfloat16)
    fekv.append_kv8(None, kd, kd, kp, vp, dev(np.asarray(slots, np.int64)))
    for pool in (kp, vp):
        got_c, got_e = codes_of(pool), exps_of(pool)
        got = ref.values(got_c, got_e)
        for i, (kept, _) in enumerate(lead):
            blk = i + 1
            e = got_e[blk].astype(int) - 127
            assert ((e >= ref.MIN_E) & (e <= ref.MAX_E)).all()
            for h in range(hkv):
                s = 2.0 ** e[h]
                want = ref.decode_e4m3(ref.encode_e4m3(before[16 * blk:16 * blk + kept, h] / s)) * s
                assert np.array_equal(got[16 * blk:16 * blk + kept, h], want)
                need = max(ref.needed(float(np.abs(k[i, h].astype(np.float64)).max())),
                           min(max(byte - 127, ref.MIN_E), ref.MAX_E))
                assert e[h] == need
    assert fekv.device_errors() == 0


# ---------------------------------------------------------------------------
# gather
# ---------------------------------------------------------------------------

def i32(*a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("kv,pages,offset", [
    ((0, 2, 4, 6), range(6), (0, 32, 65)),       # the last sequence: one row past `out`
    ((0, 2, 4, 6), range(6), (0, 32, 2 ** 30)),
    ((0, 2, 4, 6), range(6), (0, 32, -1)),
    ((0, 2, 4, 7), range(6), (0, 32, 64)),       # one page past the list
    ((0, 2, 4, 2 ** 24), range(6), (0, 32, 64)),
    ((-2, 2, 4, 6), range(6), (64, 32, 0))])     # the first sequence: before the list
def test_gather_stays_within_its_arrays(kv, pages, offset):
    """A sequence whose rows reach past `out`, or whose pages past the list,
    is skipped and flagged; the others are gathered, nothing else is written."""
    rng = np.random.default_rng(2)
    codes, exps = random_pool(rng, 8 * 16, 2, 128)
    buf = torch.full((200, 2, 128), 5.0, device="cuda", dtype=torch.float16)
    fekv.gather_kv8(pool_of(codes, exps), buf[50:146], i32(*kv), i32(*pages), i32(16, 16, 16),
                    i32(*offset), 32, 16)
    got = buf.float().cpu().numpy()
    want = np.full(got.shape, 5.0)
    val = ref.values(codes, exps)
    for b in (1, 2) if kv[0] < 0 else (0, 1):
        want[50 + offset[b]:82 + offset[b]] = val[16 * kv[b]:16 * kv[b] + 32]
    assert np.array_equal(got, half(want, False))
    assert fekv.device_errors() == _lib.FE_DEVERR_PAGE_RANGE


# ---------------------------------------------------------------------------
# attention, within the bound of each rounding that the kernels make
# ---------------------------------------------------------------------------

def check(st, causal, got=None):
    got = st.run(causal) if got is None else got
    want, bound = bounds.attention(st.q, *st.pools, st.md, st.hq, st.hkv, st.page, causal, st.bf16)
    over = np.abs(got - want) / bound
    assert np.isfinite(got).all()
    assert over.max() <= 1, (over.max(), np.unravel_index(over.argmax(), over.shape))


# ---------------------------------------------------------------------------
# plans: prepared on the device, for replay
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("hkv", [4, 3])
@pytest.mark.parametrize("bf16", [True, False])
def test_device_prepare_at_256_dims(rows, hkv, bf16):
    rng = np.random.default_rng(24)
    st = Step(rng, 4 * hkv, hkv, 256, 16, [900, 64, 333, 41], [rows] * 4, bf16)
    host, device = st.run(True), st.run(True, st.plan(device=True))
    if rows * 4 <= 16:
        assert np.array_equal(host, device)  # the same cuts
    check(st, True, device)
    check(st, False, st.run(False, st.plan(device=True)))
