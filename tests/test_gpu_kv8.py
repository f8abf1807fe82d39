"""The 8-bit KV cache on the GPU against its definition in 64 bits
(kv8_ref.py): append, gather and block copies bit for bit, attention within
the bound that its roundings give."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import fekv
import kv8_ref as ref
from fekv import _lib
from fekv.metadata import build_step_metadata

pytestmark = pytest.mark.gpu

DT = {True: torch.bfloat16, False: torch.float16}


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def pool_of(codes, exps):
    return fekv.Kv8Pool(dev(codes).view(torch.float8_e4m3fn), dev(exps))


def codes_of(pool):
    return pool.codes.view(torch.uint8).cpu().numpy()


def exps_of(pool):
    return pool.exps.cpu().numpy()


def random_pool(rng, slots, hkv, dim, spread=4):
    codes = ref.encode_e4m3(rng.standard_normal((slots, hkv, dim)) * 60)
    exps = rng.integers(127 - 8 - spread, 127 - 6 + spread, (slots // 16, hkv)).astype(np.uint8)
    return codes, exps


def half(x, bf16):
    """x rounded to the 16-bit type, as float32."""
    return torch.from_numpy(np.asarray(x, np.float32)).to(DT[bf16]).float().numpy()


def rope_cache(n, rot):
    f = 1e4 ** (-np.arange(rot // 2) / (rot // 2))
    a = np.arange(n)[:, None] * f
    return np.concatenate([np.cos(a), np.sin(a)], 1).astype(np.float32)


def same_codes(got, want):
    """Equal codes; a NaN may have either sign."""
    nan = (want & 0x7F) == 0x7F
    assert np.array_equal(got[~nan], want[~nan])
    assert ((got[nan] & 0x7F) == 0x7F).all()


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------

def run_append(rng, k, v, slots, pos, cache, pools, bf16, hq, q=None, alias=False):
    """Runs append_kv8 and the restatement on copies; compares whole pools."""
    hkv, dim = k.shape[1:]
    rows = len(slots)
    q = half(rng.standard_normal((rows, hq, dim)), bf16) if q is None else q
    (kc, ke), (vc, ve) = pools
    kp, vp = pool_of(kc, ke), pool_of(vc, ve)
    qd = dev(q, DT[bf16])
    out = qd if alias else torch.full_like(qd, 7.0)
    fekv.append_kv8(qd, dev(k, DT[bf16]), dev(v, DT[bf16]), kp, vp, dev(np.asarray(slots, np.int64)),
                    dev(np.asarray(pos, np.int64)), None if cache is None else dev(cache),
                    q_out=None if alias else out)
    torch.cuda.synchronize()
    skip = set()
    kr, qr = k, q
    if cache is not None:
        skip = {i for i, p in enumerate(pos) if not 0 <= p < cache.shape[0]}
        safe = np.array([p if 0 <= p < cache.shape[0] else 0 for p in pos])
        kr, qr = ref.rotate(k, safe, cache), ref.rotate(q, safe, cache)
    ref.append(kr, kc, ke, slots, skip)
    ref.append(v, vc, ve, slots, skip)
    same_codes(codes_of(kp), kc)
    same_codes(codes_of(vp), vc)
    assert np.array_equal(exps_of(kp), ke)
    assert np.array_equal(exps_of(vp), ve)
    want = half(qr, bf16)
    got = out.float().cpu().numpy()
    for i in skip:
        want[i] = q[i] if alias else 7.0
    assert np.array_equal(got, want, equal_nan=True)


def step_slots(rng, page, starts, counts, blocks):
    """Slots, positions of `counts[b]` tokens from position starts[b] on."""
    perm = rng.permutation(blocks)
    slots, pos, at = [], [], 0
    for s, n in zip(starts, counts):
        need = -(-(s + n) // page)
        table = perm[at:at + need]
        at += need
        t = np.arange(s, s + n)
        slots.append(table[t // page] * page + t % page)
        pos.append(t)
    return np.concatenate(slots), np.concatenate(pos)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("hq,hkv,dim,rot,page", [(16, 8, 128, 128, 16), (8, 4, 128, 64, 32),
                                                 (6, 3, 128, 0, 48), (16, 2, 256, 256, 16),
                                                 (5, 5, 256, 72, 64), (2, 1, 128, 8, 16)])
def test_append_steps_and_chunks(bf16, hq, hkv, dim, rot, page):
    rng = np.random.default_rng(hq * dim + rot)
    starts = [0, 1, 15, 16, 17, 30, 5]
    counts = [1, 1, 1, 1, 40, 2, 33]
    slots, pos = step_slots(rng, page, starts, counts, 40)
    rows = len(slots)
    k = half(rng.standard_normal((rows, hkv, dim)) * np.exp2(rng.integers(-6, 7, (rows, hkv, 1))),
             bf16)
    v = half(rng.standard_normal((rows, hkv, dim)), bf16)
    pools = [random_pool(rng, 41 * page, hkv, dim) for _ in range(2)]
    cache = rope_cache(64, rot) if rot else None
    run_append(rng, k, v, slots, pos, cache, pools, bf16, hq, alias=bf16)
    assert fekv.device_errors() == 0


@pytest.mark.parametrize("hkv,dim", [(8, 128), (8, 256)])
def test_append_many_rows(hkv, dim):
    """Enough rows that a warp covers 16 of them, starting anywhere in a block."""
    rng = np.random.default_rng(3)
    counts = [1, 2000, 16, 17, 1, 1, 2100, 3]
    starts = [9, 5, 0, 3, 15, 16, 1, 14]
    slots, pos = step_slots(rng, 16, starts, counts, 300)
    k = half(rng.standard_normal((len(slots), hkv, dim)), True)
    v = half(rng.standard_normal((len(slots), hkv, dim)), True)
    pools = [random_pool(rng, 301 * 16, hkv, dim) for _ in range(2)]
    run_append(rng, k, v, slots, pos, rope_cache(2200, dim), pools, True, 2)
    assert fekv.device_errors() == 0


@pytest.mark.parametrize("many", [False, True])
def test_append_skips_and_flags(many):
    """Padding rows, slots past the pool and positions past the table are
    skipped, and flagged where they are errors."""
    rng = np.random.default_rng(4)
    hkv, dim = (8, 128)
    n = 4200 if many else 24
    slots = np.arange(16, 16 + n)
    pos = np.arange(n) % 50
    slots[5], slots[9] = -1, 10 ** 12
    pos[13] = 50
    pos[17] = -3
    cs = (16 + n + 31) // 16 * 16
    k = half(rng.standard_normal((n, hkv, dim)), True)
    pools = [random_pool(rng, cs, hkv, dim) for _ in range(2)]
    run_append(rng, k, k, slots, pos, rope_cache(50, 128), pools, True, 3)
    assert fekv.device_errors() == _lib.FE_DEVERR_SLOT_RANGE | _lib.FE_DEVERR_POS_RANGE


@pytest.mark.parametrize("gap", [1, 14, 40, 70])
def test_append_runs_go_on_past_skipped_rows(gap):
    """A block's rows with up to 70 skipped rows among them are one run, in
    both window sizes (the second call has rows enough for 16-row windows)."""
    for more in (0, 4200):
        rng = np.random.default_rng(gap)
        slots = [16, 17, *[-1] * gap, 18, 19, *[-1] * gap, 25, 32, *[-1] * gap, 33, 40]
        slots += list(range(64, 64 + more))
        k = half(rng.standard_normal((len(slots), 8, 128)) *
                 np.exp2(rng.integers(-3, 4, (len(slots), 1, 1))), True)
        pools = [random_pool(rng, (64 + more + 31) // 16 * 16, 8, 128) for _ in range(2)]
        run_append(rng, k, k[::-1].copy(), slots, [0] * len(slots), None, pools, True, 1)
    assert fekv.device_errors() == 0


@pytest.mark.parametrize("gap", [0, 1, 2, 5, 33])
def test_append_windows_of_four_rows(gap):
    """Rows enough for 4-row windows, few enough not for 16-row ones: blocks
    begun anywhere, and blocks with skipped rows inside."""
    rng = np.random.default_rng(40 + gap)
    counts = [700, 1, 16, 17, 400, 3, 1, 900]
    starts = [9, 15, 0, 3, 16, 14, 31, 5]
    slots, pos = step_slots(rng, 16, starts, counts, 200)
    slots = np.insert(slots, 300, [-1] * gap)
    slots = np.insert(slots, 1000, [-1] * gap)
    pos = np.insert(np.insert(pos, 300, [0] * gap), 1000, [0] * gap)
    k = half(rng.standard_normal((len(slots), 8, 128)) *
             np.exp2(rng.integers(-3, 4, (len(slots), 1, 1))), True)
    pools = [random_pool(rng, 200 * 16, 8, 128) for _ in range(2)]
    run_append(rng, k, k[::-1].copy(), slots, pos, rope_cache(1000, 128), pools, True, 2)
    assert fekv.device_errors() == 0


def test_append_special_values():
    """Zeros, infinities, NaN, subnormals, the largest finite numbers, and
    magnitudes at the edge of a scale (448, 1.75 * 2^n, and just above)."""
    rng = np.random.default_rng(5)
    hkv, dim = 2, 128
    special = [0.0, np.inf, -np.inf, np.nan, 1e-40, -3e38, 448.0, 1.75, 1.7578125, 464.0, 2.0 ** -40,
               2.0 ** 100, -0.0]
    rows = len(special)
    k = np.zeros((rows, hkv, dim), np.float32)
    k[:, 1] = rng.standard_normal((rows, dim)) * 0.01
    for i, x in enumerate(special):
        k[i, :, i] = x
    v = k[::-1].copy()
    slots = np.arange(rows) * 16 + np.arange(rows)  # one block each, every offset
    pools = [random_pool(rng, 16 * rows, hkv, dim) for _ in range(2)]
    q = half(np.ones((rows, 1, dim)), True)
    run_append(rng, half(k, True), half(v, True), slots, [0] * rows, None, pools, True, 1, q=q)
    # the same values in one run
    pools = [random_pool(rng, 32, hkv, dim) for _ in range(2)]
    run_append(rng, half(k, True), half(v, True), np.arange(16, 16 + rows), [0] * rows, None, pools,
               True, 1, q=q)


def test_append_token_by_token_grows():
    """A block filled a token at a time with growing magnitudes: the kept
    tokens move to each new scale; refilling the block from its start resets."""
    rng = np.random.default_rng(6)
    hkv, dim = 8, 128
    pools = [random_pool(rng, 48, hkv, dim) for _ in range(2)]
    for rep in range(2):
        for t in range(20):
            x = half(rng.standard_normal((1, hkv, dim)) * 2.0 ** (t // 3 - rep), False)
            run_append(rng, x, x, [16 + t], [t], rope_cache(32, 128), pools, False, 8)


def test_append_nothing_and_no_queries():
    p = fekv.Kv8Pool.empty(3, 16, 2, 128)
    k = torch.zeros(0, 2, 128, device="cuda", dtype=torch.float16)
    fekv.append_kv8(None, k, k, p, p, torch.zeros(0, dtype=torch.int64, device="cuda"))
    k = torch.ones(1, 2, 128, device="cuda", dtype=torch.float16)
    p2 = fekv.Kv8Pool.empty(3, 16, 2, 128)
    fekv.append_kv8(None, k, k, p, p2, torch.full((1,), 16, dtype=torch.int64, device="cuda"))
    torch.cuda.synchronize()
    val = ref.values(codes_of(p), exps_of(p))
    assert (val[16] == 1).all() and val.sum() == 256


# ---------------------------------------------------------------------------
# gather and block copies
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("hkv,dim,page", [(8, 128, 16), (3, 128, 48), (1, 256, 16), (5, 256, 32)])
def test_gather(bf16, hkv, dim, page):
    rng = np.random.default_rng(hkv)
    lens = [1, 15, 16, 17, 300, 47, 48, 49, 2]
    tables = np.split(rng.permutation(60), np.cumsum([-(-n // page) for n in lens]))
    codes, exps = random_pool(rng, 61 * page, hkv, dim)
    codes[np.where((codes & 0x7F) == 0x7F)] = 0
    md = build_step_metadata(tables[:len(lens)], lens, [0] * len(lens), page)
    off = np.cumsum([0] + lens[:-1])
    out = torch.full((sum(lens) + 2, hkv, dim), 5.0, device="cuda", dtype=DT[bf16])
    i32 = lambda a: dev(np.asarray(a, np.int32))  # noqa: E731
    fekv.gather_kv8(pool_of(codes, exps), out[1:], i32(md.kv), i32(md.pages), i32(md.last), i32(off),
                    max(lens), page)
    got = out.float().cpu().numpy()
    val = ref.values(codes, exps)
    want = np.concatenate([val[np.asarray(t)[np.arange(n) // page] * page + np.arange(n) % page]
                           for t, n in zip(tables, lens)])
    assert np.array_equal(got[1:-1], half(want, bf16))
    assert (got[0] == 5).all() and (got[-1] == 5).all()
    assert fekv.device_errors() == 0


def test_gather_bad_page_is_skipped():
    pool = fekv.Kv8Pool.empty(3, 16, 2, 128)
    out = torch.full((32, 2, 128), 5.0, device="cuda", dtype=torch.float16)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    fekv.gather_kv8(pool, out, i32(0, 2), i32(1, 77), i32(16), i32(0), 32, 16)
    assert (out[:16] == 0).all() and (out[16:] == 5).all()
    assert fekv.device_errors() == _lib.FE_DEVERR_PAGE_RANGE


def test_gather_bad_last_skips_its_sequence():
    pool = fekv.Kv8Pool.empty(7, 16, 2, 128)
    out = torch.full((6 * 16, 2, 128), 5.0, device="cuda", dtype=torch.float16)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    fekv.gather_kv8(pool, out, i32(0, 2, 4, 4, 6), i32(0, 1, 2, 3, 4, 5), i32(17, 16, 9, 0),
                    i32(0, 32, 0, 64), 32, 16)
    assert (out[:32] == 5).all() and (out[32:64] == 0).all() and (out[64:] == 5).all()
    assert fekv.device_errors() == _lib.FE_DEVERR_PAGE_RANGE


@pytest.mark.parametrize("hkv,dim,page,layers", [(8, 128, 16, 1), (3, 128, 48, 5), (2, 256, 32, 3)])
def test_copy_blocks(hkv, dim, page, layers):
    rng = np.random.default_rng(page)
    pages = 20
    perm = rng.permutation(pages)
    ntok = [0, 1, page, page - 1, 16, 15, page // 2]
    src, dst = perm[:7], perm[7:14]
    pools = [[random_pool(rng, (pages + 1) * page, hkv, dim) for _ in range(layers)]
             for _ in range(2)]
    d = [[pool_of(*p) for p in side] for side in pools]
    i32 = lambda a: dev(np.asarray(a, np.int32))  # noqa: E731
    # two entries that must be skipped and flagged
    fekv.copy_blocks_kv8(d[0], d[1], i32([*src, pages + 1, 3]), i32([*dst, 2, 4]),
                         i32([*ntok, 4, page + 1]), page)
    for side, got in zip(pools, d):
        for (codes, exps), g in zip(side, got):
            c = codes.reshape(pages + 1, page, hkv, dim)
            e = exps.reshape(pages + 1, page // 16, hkv)
            for a, b, n in zip(src, dst, ntok):
                c[b, :n] = c[a, :n]
                e[b, :-(-n // 16)] = e[a, :-(-n // 16)]
            assert np.array_equal(codes_of(g), codes)
            assert np.array_equal(exps_of(g), exps)
    assert fekv.device_errors() == _lib.FE_DEVERR_PAGE_RANGE | _lib.FE_DEVERR_NTOK_RANGE


def test_fork_lists_drive_copies():
    """fork_copies' lists, a partial tail: parent and child read the same
    prefix and then append on their own."""
    rng = np.random.default_rng(8)
    page, hkv, dim, n = 16, 4, 128, 37
    kc, ke = random_pool(rng, 8 * page, hkv, dim)
    parent, child = [5, 2, 6], [5, 2, 0]
    src, dst, ntok = fekv.fork_copies([parent], [child], [n], page)
    kp, vp = pool_of(kc, ke), pool_of(kc, ke)
    fekv.copy_blocks_kv8([kp], [vp], dev(src), dev(dst), dev(ntok), page)
    got = ref.values(codes_of(kp), exps_of(kp))
    t = np.arange(n)
    a, b = (np.asarray(x)[t // page] * page + t % page for x in (parent, child))
    assert np.array_equal(got[a], got[b])


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

class Step:
    """A prepared step over random pools; every slot outside the sequences
    holds NaN codes, and blocks without a token absurd exponents."""

    def __init__(self, rng, hq, hkv, dim, page, lens, rows, bf16, blocks=None, spread=4):
        need = [-(-n // page) for n in lens]
        self.blocks = sum(need) + 3 if blocks is None else blocks
        perm = rng.permutation(self.blocks)
        tables = np.split(perm[:sum(need)], np.cumsum(need)[:-1])
        self.md = build_step_metadata(tables, [n - r for n, r in zip(lens, rows)], rows, page)
        self.hq, self.hkv, self.dim, self.page, self.bf16 = hq, hkv, dim, page, bf16
        slots = (self.blocks + 1) * page
        used = np.zeros(slots, bool)
        for t, n in zip(tables, lens):
            i = np.arange(n)
            used[np.asarray(t)[i // page] * page + i % page] = True
        self.used = used
        self.pools = []
        for _ in range(2):
            codes, exps = random_pool(rng, slots, hkv, dim, spread)
            codes[~used] = 0x7F
            empty = ~used.reshape(-1, 16).any(1)
            exps[empty] = rng.choice([0, 255], (int(empty.sum()), 1))
            self.pools.append((codes, exps))
        self.q = half(rng.standard_normal((sum(rows), hq, dim)), bf16)

    def plan(self, device=False):
        md = self.md
        p = fekv.Kv8Plan(self.hq, self.hkv, self.dim, self.page, md.batch,
                         int((md.kv[1:] - md.kv[:-1]).max()), self.bf16, self.blocks)
        if device:
            i32 = lambda a: dev(np.asarray(a, np.int32))  # noqa: E731
            p.prepare_device(i32(md.qo), i32(md.kv), i32(md.pages), i32(md.last), md.batch, md.rows)
        else:
            p.prepare(md.qo, md.kv, md.pages, md.last)
        return p

    def run(self, causal, plan=None):
        plan = self.plan() if plan is None else plan
        qd = dev(self.q, DT[self.bf16])
        out = torch.full_like(qd, 9.0)
        plan.attention(qd, pool_of(*self.pools[0]), pool_of(*self.pools[1]), out, causal)
        torch.cuda.synchronize()
        assert fekv.device_errors() == 0
        plan.close()
        return out.double().cpu().numpy()

    def expect(self, causal):
        k, v = (ref.values(*p) for p in self.pools)
        return ref.attention(self.q.astype(np.float64), k, v, self.md, self.hq, self.hkv, self.page,
                             causal, self.bf16)

    def check(self, causal, got=None):
        got = self.run(causal) if got is None else got
        want, bound = self.expect(causal)
        over = np.abs(got - want) - bound
        assert np.isfinite(got).all()
        assert over.max() <= 0, (over.max(), np.unravel_index(over.argmax(), over.shape))


HEADS = [(16, 8, 128, 16), (32, 4, 128, 32), (12, 12, 128, 16), (6, 3, 128, 48), (10, 2, 128, 16),
         (16, 1, 128, 16), (16, 2, 256, 16), (4, 4, 256, 32), (15, 3, 256, 16)]


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("hq,hkv,dim,page", HEADS)
def test_decode(bf16, hq, hkv, dim, page):
    rng = np.random.default_rng(hq + hkv)
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 500, 1, 700]
    Step(rng, hq, hkv, dim, page, lens, [1] * len(lens), bf16).check(True)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hq,hkv,dim,page", HEADS)
def test_multi_row(hq, hkv, dim, page, causal):
    """Verify blocks, chunks that start a sequence, chunks over a prefix, rows
    and keys that end inside a tile, decode rows beside them."""
    rng = np.random.default_rng(hq * hkv + dim)
    lens = [2, 16, 40, 129, 300, 64, 140, 1, 33, 128]
    rows = [2, 16, 5, 129, 17, 64, 40, 1, 1, 127]
    bf16 = causal
    Step(rng, hq, hkv, dim, page, lens, rows, bf16).check(causal)


@pytest.mark.parametrize("dim", [128, 256])
def test_one_long_sequence_is_cut(dim):
    """One sequence, few rows, many keys: its row items' keys are cut across
    CTAs and joined."""
    rng = np.random.default_rng(dim)
    st = Step(rng, 8, 2, dim, 16, [6000, 3001], [9, 30], True)
    p = st.plan()
    assert p.info()["split_sequences"] > 0
    st.check(True, st.run(True, p))
    st.check(False)


@pytest.mark.parametrize("rows", [1, 20])
@pytest.mark.parametrize("dim", [128, 256])
def test_small_weights_keep_their_share(rows, dim):
    """A first key that takes nearly all of the softmax and has no value, and
    thousands of keys 2^-20 below it: the output is those keys' alone."""
    rng = np.random.default_rng(9)
    n = 5000
    st = Step(rng, 4, 2, dim, 16, [n], [rows], True, spread=0)
    (kc, ke), (vc, ve) = st.pools
    ke[:], ve[:] = 127 - 6, 127 - 6
    slot = int(st.md.pages[0]) * 16
    st.q[:] = 0.0
    kc[st.used, :, 0] = 0
    want = np.log(2.0 ** 20) * np.sqrt(dim) * 2.0 ** 6
    kc[slot, :, 0] = ref.encode_e4m3(np.full(2, want / 64))
    st.q[..., 0] = 64.0
    vc[slot] = 0
    st.check(True)


def test_block_scales_far_apart():
    """V scales that differ by 2^40 between blocks, blocks of zeros, and K
    scales that differ by 2^6."""
    for rows, dim in [(1, 128), (1, 256), (24, 128), (24, 256)]:
        rng = np.random.default_rng(rows + dim)
        st = Step(rng, 8, 2, dim, 16, [700, 300], [rows, rows], True)
        (kc, ke), (vc, ve) = st.pools
        ve[:] = 127 + rng.integers(-30, 10, ve.shape)
        ke[:] = 127 + rng.integers(-13, -6, ke.shape)
        zero = rng.random(ve.shape) < 0.3
        vc.reshape(-1, 16, *vc.shape[1:])[zero.nonzero()[0], :, zero.nonzero()[1]] = 0
        ve[zero] = 127 - 32
        st.check(True)


@pytest.mark.parametrize("rows", [1, 40])
def test_queries_of_any_size(rows):
    """Zero rows, tiny and huge rows, rows with an outlier; rows that hold NaN
    or infinity give NaN and touch no other."""
    rng = np.random.default_rng(rows)
    st = Step(rng, 8, 2, 128, 16, [200, 77], [rows, rows], True)
    st.q[0, 0] = 0
    st.q[0, 1] *= 1e-30
    st.q[0, 2, 5] *= 1000
    st.q[0, 3] *= 2.0 ** 5
    st.q = half(st.q, True)
    st.check(True)
    st.q[-1, 0, 3] = np.nan
    st.q[-1, 5, 100] = np.inf
    got = st.run(True)
    assert np.isnan(got[-1, 0]).all() and np.isnan(got[-1, 5]).all()
    got[-1, [0, 5]] = 0
    st.q[-1, [0, 5]] = 0
    want, bound = st.expect(True)
    want[-1, [0, 5]] = 0
    assert (np.abs(got - want) <= bound).all()


def test_nan_in_a_key_or_value_stays_in_its_head():
    rng = np.random.default_rng(12)
    st = Step(rng, 8, 4, 128, 16, [50, 60], [1, 20], True)
    clean = st.run(True)
    (kc, _), (vc, _) = st.pools
    kc[int(st.md.pages[0]) * 16 + 3, 1, 7] = 0x7F
    vc[int(st.md.pages[4]) * 16 + 3, 2, 9] = 0xFF
    got = st.run(True)
    assert np.isnan(got[0, 2:4]).all()
    assert np.isnan(got[1:, 4:6, 9]).all()
    got[0, 2:4] = clean[0, 2:4]
    got[1:, 4:6, 9] = clean[1:, 4:6, 9]
    assert np.array_equal(got, clean)


def test_offsets_past_32_bits():
    """A pool of more than 2^32 codes, the sequences in its last pages."""
    hq, hkv, dim, page = 8, 8, 256, 16
    rng = np.random.default_rng(13)
    blocks = 2 ** 32 // (page * hkv * dim) + 40
    st = Step(rng, hq, hkv, dim, page, [100, 70, 200], [1, 1, 30], True)
    shift = blocks - st.blocks
    slots = (blocks + 1) * page
    pools = []
    for codes, exps in st.pools:
        c = torch.zeros(slots, hkv, dim, dtype=torch.uint8, device="cuda")
        e = torch.zeros(slots // 16, hkv, dtype=torch.uint8, device="cuda")
        c[shift * page:] = dev(codes)
        e[shift * page // 16:] = dev(exps)
        pools.append(fekv.Kv8Pool(c.view(torch.float8_e4m3fn), e))
    md = st.md
    plan = fekv.Kv8Plan(hq, hkv, dim, page, md.batch, 20, True, blocks)
    plan.prepare(md.qo, md.kv, md.pages + shift, md.last)
    qd = dev(st.q, torch.bfloat16)
    out = torch.empty_like(qd)
    plan.attention(qd, *pools, out, True)
    torch.cuda.synchronize()
    plan.close()
    st.check(True, out.double().cpu().numpy())
    # append and gather there
    slot = slots - 16 + 3
    k = torch.randn(1, hkv, dim, device="cuda", dtype=torch.bfloat16)
    fekv.append_kv8(None, k, k, *pools, torch.tensor([slot], device="cuda"))
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    got = torch.empty(4, hkv, dim, device="cuda", dtype=torch.bfloat16)
    fekv.gather_kv8(pools[0], got, i32(0, 1), i32(blocks), i32(4), i32(0), 4, page)
    c, e = pools[0].codes[slot].view(torch.uint8).cpu().numpy(), pools[0].exps[-1].cpu().numpy()
    val = ref.decode_e4m3(c) * np.exp2(e.astype(float) - 127)[:, None]
    assert np.array_equal(got[3].double().cpu().numpy(), val)
    assert fekv.device_errors() == 0


# ---------------------------------------------------------------------------
# plans, streams, graphs
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("rows", [1, 3, 40])
def test_device_prepare_gives_the_same_bits(rows):
    rng = np.random.default_rng(14)
    st = Step(rng, 16, 4, 128, 16, [900, 64, 333, 41], [rows] * 4, True)
    host, device = st.run(True), st.run(True, st.plan(device=True))
    if rows * 4 <= 16:
        assert np.array_equal(host, device)  # the same cuts
    st.check(True, device)


def test_a_step_replays_from_a_graph():
    """Device-side prepare, append and attention captured once; a second step
    replays with other tables, starts, queries and keys, on another stream."""
    rng = np.random.default_rng(15)
    hq, hkv, dim, page, batch, rows = 8, 4, 128, 16, 3, 2
    blocks = 60
    tables = dev(rng.permutation(blocks)[:batch * 16].reshape(batch, 16).astype(np.int32))
    starts = torch.zeros(batch, dtype=torch.int32, device="cuda")
    slots = torch.zeros(batch * rows, dtype=torch.int64, device="cuda")
    pos = torch.zeros_like(slots)
    q = torch.zeros(batch * rows, hq, dim, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(batch * rows, hkv, dim, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    qr, out = torch.zeros_like(q), torch.zeros_like(q)
    cache = rope_cache(300, 128)
    rope = dev(cache)
    pools = [pool_of(*random_pool(rng, (blocks + 1) * page, hkv, dim)) for _ in range(2)]
    plan = fekv.Kv8Plan(hq, hkv, dim, page, batch, 16, True, blocks)

    def step():
        plan.step_prepare_device(tables, starts, rows, slots, pos)
        fekv.append_kv8(q, k, v, *pools, slots, pos, rope, q_out=qr)
        plan.attention(qr, *pools, out, True)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        for first in ([5, 100, 31], [7, 102, 33]):
            starts.copy_(dev(np.asarray(first, np.int32)))
            for t in (q, k, v):
                t.copy_(torch.randn(t.shape, device="cuda"))
            graph.replay()
            side.synchronize()
            md = build_step_metadata(list(tables.cpu().numpy()), first, [rows] * batch, page)
            assert np.array_equal(slots.cpu().numpy(), md.slots)
            kv = [ref.values(codes_of(p), exps_of(p)) for p in pools]
            want, bound = ref.attention(qr.double().cpu().numpy(), *kv, md, hq, hkv, page, True,
                                        True)
            assert (np.abs(out.double().cpu().numpy() - want) <= bound).all()
    assert fekv.device_errors() == 0
    plan.close()


def test_mixed_step_beside_each_other():
    """Long chunks and enough decode rows that the plan runs its two kernels
    side by side."""
    rng = np.random.default_rng(16)
    lens = [600] * 4 + [int(x) for x in rng.integers(900, 1600, 40)]
    st = Step(rng, 16, 4, 128, 16, lens, [300] * 4 + [1] * 40, True)
    st.check(True)


def test_plans_do_not_mix():
    a = fekv.Kv8Plan(8, 4, 128, 16, 1, 4, True, 8)
    b = fekv.AttentionPlan(8, 4, 128, 16, 1, 4, True, 8)
    for p in (a, b):
        p.prepare([0, 1], [0, 1], [2], [5])
    q = torch.zeros(1, 8, 128, dtype=torch.bfloat16, device="cuda")
    kv = torch.zeros(144, 4, 128, dtype=torch.bfloat16, device="cuda")
    pool = fekv.Kv8Pool.empty(8, 16, 4, 128)
    with pytest.raises(fekv.FeError) as e:
        fekv.AttentionPlan.attention(a, q, kv, kv, q)
    assert e.value.status == _lib.FE_ERR_INVALID_ARGUMENT
    with pytest.raises(fekv.FeError) as e:
        _attention_on(b, q, pool)
    assert e.value.status == _lib.FE_ERR_INVALID_ARGUMENT
    a.close()
    b.close()


def _attention_on(plan, q, pool):
    ptr = lambda t: t.data_ptr()  # noqa: E731
    _lib.check(plan.lib.fe_kv8_attn_run(plan.handle, ptr(q), ptr(pool.codes), ptr(pool.codes),
                                        ptr(pool.exps), ptr(pool.exps), ptr(q), 1, None),
               "attention")


def test_python_refusals():
    pool = fekv.Kv8Pool.empty(8, 16, 4, 128)
    plan = fekv.Kv8Plan(8, 4, 128, 16, 1, 4, True, 8)
    plan.prepare([0, 1], [0, 1], [2], [5])
    q = torch.zeros(1, 8, 128, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(1, 4, 128, dtype=torch.bfloat16, device="cuda")
    slots = torch.zeros(1, dtype=torch.int64, device="cuda")
    bad = [
        lambda: plan.attention(q.half(), pool, pool, q),
        lambda: plan.attention(q, pool, pool, q.float()),
        lambda: plan.attention(q[:, ::2], pool, pool, q),
        lambda: plan.attention(q, fekv.Kv8Pool.empty(9, 16, 4, 128), pool, q),
        lambda: plan.attention(q, *[fekv.Kv8Pool.empty(9, 16, 4, 128)] * 2, q),
        lambda: fekv.append_kv8(q, k.half(), k, pool, pool, slots),
        lambda: fekv.append_kv8(q, k, k[:, :2], pool, pool, slots),
        lambda: fekv.append_kv8(q, k, k, pool, pool, slots.int()),
        lambda: fekv.append_kv8(q, k, k, pool, pool, slots, None, torch.zeros(4, 128).cuda()),
        lambda: fekv.append_kv8(q, k, k, pool, pool, slots, slots, torch.zeros(4, 128)),
        lambda: fekv.append_kv8(q, k, k, pool, pool, slots, q_out=q[:, :4]),
        lambda: fekv.append_kv8(q, k, k.transpose(1, 2).contiguous().transpose(1, 2), pool, pool,
                                slots),
        lambda: fekv.Kv8Pool(pool.codes.view(torch.uint8), pool.exps),
        lambda: fekv.Kv8Pool(pool.codes, pool.exps[:-1]),
        lambda: fekv.Kv8Pool(pool.codes[:, :2], pool.exps[:, :2]),
        lambda: fekv.Kv8Pool(pool.codes.cpu(), pool.exps.cpu()),
        lambda: fekv.copy_blocks_kv8([pool], [], slots, slots, slots, 16),
        lambda: fekv.copy_blocks_kv8([pool], [pool], slots, slots, slots, 16),
        lambda: fekv.gather_kv8(pool, k, slots, slots, slots, slots, 1, 16),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    plan.close()


def test_refusals_of_short_arrays():
    pool = fekv.Kv8Pool.empty(8, 16, 4, 128)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    out = torch.zeros(16, 4, 128, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros(5, 8, 128, dtype=torch.bfloat16, device="cuda")
    for prepare in ("host", "device"):
        plan = fekv.Kv8Plan(8, 4, 128, 16, 2, 4, True, 8)
        meta = ([0, 4, 5], [0, 1, 2], [2, 3], [5, 16])
        if prepare == "host":
            plan.prepare(*meta)
        else:
            plan.prepare_device(*(i32(*m) for m in meta), 2, 5)
        with pytest.raises(ValueError):
            plan.attention(q[:4], pool, pool, q[:4])
        plan.attention(q, pool, pool, torch.empty_like(q))
        plan.close()
    for f in (lambda: fekv.gather_kv8(pool, out, i32(0, 1), i32(2), i32(5, 6), i32(0), 16, 16),
              lambda: fekv.gather_kv8(pool, out, i32(0, 1), i32(2), i32(5), i32(0, 0), 16, 16),
              lambda: fekv.copy_blocks_kv8([pool], [pool], i32(1, 2), i32(3), i32(4, 4), 16),
              lambda: fekv.copy_blocks_kv8([pool], [pool], i32(1), i32(3), i32(), 16)):
        with pytest.raises(ValueError):
            f()
    assert fekv.device_errors() == 0
