"""Forms of the 8-bit cache's operators that test_gpu_kv8.py does not reach,
against the same restatement in 64 bits (kv8_ref.py)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import fekv
import kv8_bounds as bounds
import kv8_ref as ref
from fekv import _lib
from fekv.metadata import build_step_metadata
from test_gpu_kv8 import (HEADS, Step, codes_of, dev, exps_of, half, pool_of, random_pool,
                          rope_cache, run_append, step_slots)

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


# Rows times heads choose the append's form: up to 2 Ki pairs K and V have warps
# of their own, up to 8 Ki they share one, then windows of 4 rows, from 32 Ki 16.
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("hkv,dim,rot,rows", [
    (8, 128, 128, 150), (8, 128, 64, 600), (8, 128, 128, 900), (8, 128, 128, 1500),
    (8, 128, 0, 4300), (8, 128, 128, 4300), (4, 256, 256, 300), (4, 256, 64, 900),
    (4, 256, 128, 2600), (4, 256, 0, 2600), (4, 256, 256, 8400), (3, 128, 128, 1100)])
def test_append_forms(bf16, hkv, dim, rot, rows):
    """Each form in both types and at both widths: blocks begun anywhere, kept
    tokens whose scale grows, skipped rows inside a block, whole blocks."""
    rng = np.random.default_rng(rows + dim + bf16)
    counts = [1, rows // 2, 16, 17, 1, 3, rows - rows // 2]
    starts = [9, 5, 0, 3, 15, 14, 31]
    slots, pos = step_slots(rng, 16, starts, counts, rows // 16 + 40)
    for at, gap in ((40, 3), (60, 1), (100, 20)):
        slots, pos = (np.insert(a, at, [x] * gap) for a, x in ((slots, -1), (pos, 0)))
    k = half(rng.standard_normal((len(slots), hkv, dim)) *
             np.exp2(rng.integers(-4, 5, (len(slots), 1, 1))), bf16)
    pools = [random_pool(rng, (rows // 16 + 41) * 16, hkv, dim) for _ in range(2)]
    cache = rope_cache(int(pos.max()) + 1, rot) if rot else None
    run_append(rng, k, k[::-1].copy(), slots, pos, cache, pools, bf16, 3)
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


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hq,hkv,dim,page", HEADS)
def test_multi_row(hq, hkv, dim, page, causal, bf16):
    """Verify blocks, chunks that start a sequence, chunks over a prefix, rows
    and keys that end inside a tile, decode rows beside them."""
    rng = np.random.default_rng(hq * hkv + dim + 7)
    lens = [2, 16, 40, 129, 300, 64, 140, 1, 33, 128, 700]
    rows = [2, 16, 5, 129, 17, 64, 40, 1, 1, 127, 1]
    check(Step(rng, hq, hkv, dim, page, lens, rows, bf16), causal)


@pytest.mark.parametrize("rows", [1, 20])
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("bf16", [True, False])
def test_every_part_of_a_query_counts(bf16, dim, rows):
    """Scores that come from the queries' last bits alone: all else cancels."""
    rng = np.random.default_rng(rows + dim)
    st = Step(rng, 8, 4, dim, 16, [300, 40, 77], [rows] * 3, bf16)
    st.q = half(bounds.cancelling_queries(rng, 3 * rows, 8, dim, bf16), bf16)
    bounds.even_keys(rng, *st.pools[0], dim, bf16)
    st.pools[0][0][~st.used] = 0x7F
    check(st, True)
    check(st, False)


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("bf16", [True, False])
def test_long_sequences_are_cut(dim, bf16):
    """Few rows, many keys: the row items' keys are cut across CTAs and joined."""
    rng = np.random.default_rng(dim + 1)
    st = Step(rng, 8, 2, dim, 16, [6000, 3001], [9, 30], bf16)
    p = st.plan()
    assert p.info()["split_sequences"] > 0
    check(st, True, st.run(True, p))
    check(st, False)


@pytest.mark.parametrize("rows,dim", [(1, 128), (1, 256), (24, 128), (24, 256)])
@pytest.mark.parametrize("bf16", [True, False])
def test_block_scales_far_apart(rows, dim, bf16):
    """V scales that differ by 2^40 between blocks, blocks of zeros, and K
    scales that differ by 2^6."""
    rng = np.random.default_rng(rows + dim + 1)
    st = Step(rng, 8, 2, dim, 16, [700, 300], [rows, rows], bf16)
    (kc, ke), (vc, ve) = st.pools
    ve[:] = 127 + rng.integers(-30, 3, ve.shape)
    ke[:] = 127 + rng.integers(-13, -6, ke.shape)
    zero = rng.random(ve.shape) < 0.3
    vc.reshape(-1, 16, *vc.shape[1:])[zero.nonzero()[0], :, zero.nonzero()[1]] = 0
    ve[zero] = 127 - 32
    check(st, True)
    check(st, False)


@pytest.mark.parametrize("rows,dim", [(1, 128), (40, 128), (40, 256)])
@pytest.mark.parametrize("bf16", [True, False])
def test_queries_of_any_size(rows, dim, bf16):
    """Zero rows, tiny rows (f16: subnormal), large ones, rows with an outlier;
    rows that hold NaN or infinity give NaN and touch no other."""
    rng = np.random.default_rng(rows + dim)
    st = Step(rng, 8, 2, dim, 16, [200, 77], [rows, rows], bf16)
    st.q[0, 0] = 0
    st.q[0, 1] *= 1e-30 if bf16 else 1e-6
    st.q[0, 2, 5] *= 1000
    st.q[0, 3] *= 2.0 ** 5
    st.q[0, 4, 77] = 3e4
    st.q = half(st.q, bf16)
    for causal in (True, False):
        check(st, causal)
    clean = st.run(True)
    st.q[-1, 0, 3] = np.nan
    st.q[-1, 5, 100] = np.inf
    st.q[0, 7, 0] = -np.inf
    got = st.run(True)
    for r, h in ((-1, 0), (-1, 5), (0, 7)):
        assert np.isnan(got[r, h]).all()
        got[r, h] = clean[r, h]
    assert np.array_equal(got, clean)


def half_ulp(x, bf16):
    mant, low = (7, -126) if bf16 else (10, -14)
    return np.exp2(np.floor(np.log2(np.maximum(x, 2.0 ** low))) - mant - 1)


@pytest.mark.parametrize("rows,dim", [(1, 128), (1, 256), (3, 256), (40, 128), (40, 256)])
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("size", [1e4, 1e6, 3e6, 1e7, 1e9, 1e13])
def test_scores_of_any_size(size, bf16, rows, dim):
    """Scores far apart in fp32: one key above all others by an eighth of its
    score is the whole output, keys of one score share it evenly, however large
    the scores, of either sign."""
    rng = np.random.default_rng(rows + dim)
    for sign in (1.0, -1.0):
        st = Step(rng, 8, 2, dim, 16, [700, 41, 130], [rows] * 3, bf16)
        (kc, ke), (vc, ve) = st.pools
        st.q[:] = sign
        e = int(np.floor(np.log2(size / dim ** 0.5 / 14)))
        ke[:] = 127 + e
        kc[st.used] = ref.encode_e4m3(rng.integers(8, 13, (int(st.used.sum()), 2)) * 1.0)[..., None]
        first = [int(st.md.pages[p]) * 16 for p in st.md.kv[:-1]]
        kc[first] = ref.encode_e4m3(np.array(14.0 if sign > 0 else 6.0))
        got = st.run(True)
        for b, at in enumerate(first):
            want = np.repeat(ref.values(vc, ve)[at], 4, 0)  # [hq, dim]
            # the weight's rounding to a half, the quotient's, the result's
            near = np.abs(want) * (2.0 ** -11 + 2.0 ** -22)
            near = near + half_ulp(np.abs(want) + near, bf16)
            assert (np.abs(got[b * rows:(b + 1) * rows] - want) <= near).all()
        # one score for all keys, one scale for all values
        kc[st.used] = ref.encode_e4m3(np.array(11.0))
        ve[:] = 127 - 7
        got = st.run(True)
        want, mass = np.zeros(got.shape), np.zeros(got.shape)
        val = ref.values(vc, ve)
        for b, n in enumerate((700, 41, 130)):
            t = np.arange(n)
            slots = st.md.pages[st.md.kv[b]:st.md.kv[b + 1]][t // 16] * 16 + t % 16
            for i in range(rows):
                v = val[slots[:n - rows + i + 1]]
                want[b * rows + i] = np.repeat(v.mean(0), 4, 0)
                mass[b * rows + i] = np.repeat(np.abs(v).mean(0), 4, 0)
        # sums in fp32 over 700 keys and the quotient, weights as halves, the result
        bound = (701 * 2.0 ** -23 + 2.0 ** -11) * mass
        assert (np.abs(got - want) <= bound + half_ulp(np.abs(want) + bound, bf16)).all()


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("dim", [128, 256])
def test_nan_past_a_chunks_limit_stays_out_of_earlier_rows(dim, bf16):
    """A NaN in a chunk's last key: hidden from every row but the last, whose
    heads of that KV head it reaches."""
    rng = np.random.default_rng(dim)
    st = Step(rng, 8, 4, dim, 16, [190], [40], bf16)
    clean = st.run(True)
    st.pools[0][0][int(st.md.pages[189 // 16]) * 16 + 189 % 16, 2, 9] = 0x7F
    got = st.run(True)
    assert np.isnan(got[-1, 4:6]).all()
    got[-1, 4:6] = clean[-1, 4:6]
    assert np.array_equal(got, clean)


@pytest.mark.parametrize("bf16", [True, False])
def test_a_call_repeats_its_bits(bf16):
    """Nothing depends on the order in which CTAs or warps run."""
    rng = np.random.default_rng(21)
    lens = [600] * 3 + [5000] + [int(x) for x in rng.integers(900, 1600, 30)]
    st = Step(rng, 16, 4, 128, 16, lens, [300] * 3 + [20] + [1] * 30, bf16)
    plan = st.plan()
    pools = [pool_of(*p) for p in st.pools]
    qd = dev(st.q, DT[bf16])
    outs = [torch.full_like(qd, 9.0) for _ in range(12)]
    for o in outs:
        plan.attention(qd, *pools, o, True)
    torch.cuda.synchronize()
    for o in outs[1:]:
        assert torch.equal(o, outs[0])
    check(st, True, outs[0].double().cpu().numpy())
    plan.close()


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


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_a_device_prepared_long_block(dim, causal):
    """One block of 32 rows over thousands of keys, its items whole."""
    st = Step(np.random.default_rng(26), 8, 2, dim, 16, [5003], [32], True)
    check(st, causal, st.run(causal, st.plan(device=True)))


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("bf16", [True, False])
def test_a_host_plan_for_replay(dim, bf16):
    """prepare(graph=True): one captured call serves steps of the same batch and
    rows, decode rows, blocks and chunks, few keys and many."""
    rng = np.random.default_rng(dim)
    rows = [1, 30, 1, 5, 100]
    steps = [Step(rng, 8, 2, dim, 16, lens, rows, bf16, blocks=900)
             for lens in ([40, 33, 1, 7, 150], [3000, 4000, 17, 900, 100], [1, 30, 800, 5, 2100])]
    plan = fekv.Kv8Plan(8, 2, dim, 16, len(rows), 300, bf16, 900)
    q = dev(steps[0].q, DT[bf16])
    out = torch.zeros_like(q)
    pools = [pool_of(*p) for p in steps[0].pools]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        for i, st in enumerate(steps):
            md = st.md
            plan.prepare(md.qo, md.kv, md.pages, md.last, graph=True)
            q.copy_(dev(st.q, DT[bf16]))
            for pool, (codes, exps) in zip(pools, st.pools):
                pool.codes.view(torch.uint8).copy_(dev(codes))
                pool.exps.copy_(dev(exps))
            if i == 0:
                plan.attention(q, *pools, out, True)
                side.synchronize()
                with torch.cuda.graph(graph, stream=side):
                    plan.attention(q, *pools, out, True)
            out.fill_(9.0)
            graph.replay()
            side.synchronize()
            check(st, True, out.double().cpu().numpy())
    assert fekv.device_errors() == 0
    plan.close()


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("bf16", [True, False])
def test_a_step_of_blocks_replays_from_a_graph(dim, bf16):
    """Device-side prepare, append and attention of 20 packed rows a sequence
    captured once, a padding entry among them; replayed with other starts,
    tables and contents."""
    rng = np.random.default_rng(25)
    hq, hkv, page, batch, rows = 8, 2, 16, 4, 5
    blocks = 100
    tables = torch.zeros(batch, 20, dtype=torch.int32, device="cuda")
    starts = torch.zeros(batch, dtype=torch.int32, device="cuda")
    slots = torch.zeros(batch * rows, dtype=torch.int64, device="cuda")
    pos = torch.zeros_like(slots)
    q = torch.zeros(batch * rows, hq, dim, dtype=DT[bf16], device="cuda")
    k = torch.zeros(batch * rows, hkv, dim, dtype=DT[bf16], device="cuda")
    v = torch.zeros_like(k)
    qr, out = torch.zeros_like(q), torch.zeros_like(q)
    rope = dev(rope_cache(320, 128))
    pools = [pool_of(*random_pool(rng, (blocks + 1) * page, hkv, dim)) for _ in range(2)]
    plan = fekv.Kv8Plan(hq, hkv, dim, page, batch, 20, bf16, blocks)

    def step():
        plan.step_prepare_device(tables, starts, rows, slots, pos)
        fekv.append_kv8(q, k, v, *pools, slots, pos, rope, q_out=qr)
        plan.attention(qr, *pools, out, True)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        tables.copy_(dev(rng.permutation(blocks)[:batch * 20].reshape(batch, 20).astype(np.int32)))
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        for first in ([5, 300, 31, 0], [10, 305, 36, 5], [100, 7, -1, 250]):
            starts.copy_(dev(np.asarray(first, np.int32)))
            for t in (q, k, v):
                t.copy_(torch.randn(t.shape, device="cuda"))
            graph.replay()
            side.synchronize()
            live = [b for b in range(batch) if first[b] >= 0]
            at = np.concatenate([np.arange(b * rows, (b + 1) * rows) for b in live])
            md = build_step_metadata([tables[b].cpu().numpy() for b in live],
                                     [first[b] for b in live], [rows] * len(live), page)
            assert np.array_equal(slots.cpu().numpy()[at], md.slots)
            want, bound = bounds.attention(qr.double().cpu().numpy()[at],
                                           *[(codes_of(p), exps_of(p)) for p in pools], md, hq,
                                           hkv, page, True, bf16)
            assert (np.abs(out.double().cpu().numpy()[at] - want) <= bound).all()
    assert fekv.device_errors() == 0
    plan.close()
