"""Selection by score and compaction of the paged cache: equal to the
restatement token by token (evict_ref), bits and indexes."""
import numpy as np
import pytest

import evict_ref as ref

pytestmark = pytest.mark.gpu


def i32(v):
    import torch
    return torch.tensor(np.asarray(v, np.int32), device="cuda")


def layout(lens, page, seed, spare=2):
    """Block tables of random pages, and the pool's slots."""
    rng = np.random.default_rng(seed)
    need = [-(-n // page) for n in lens]
    order = rng.permutation(sum(need) + spare)
    at = np.cumsum([0] + need)
    return [order[a:b] for a, b in zip(at, at[1:])], (sum(need) + spare + 1) * page


def lists(tables, lens, page):
    return (i32(np.cumsum([0] + [len(t) for t in tables])), i32(np.concatenate(tables)),
            i32([(n - 1) % page + 1 for n in lens]))


def run_select(scores, tables, lens, page, budget, sink, recent, max_len=None):
    import fekv
    import torch
    kept = torch.full((len(lens), scores.shape[0], budget), 77, dtype=torch.int32, device="cuda")
    fekv.select_tokens(torch.from_numpy(scores).cuda(), *lists(tables, lens, page), kept, page,
                       max(lens) if max_len is None else max_len, sink=sink, recent=recent)
    assert fekv.device_errors() == 0
    return kept.cpu().numpy()


SELECT = [  # lens, page, hkv, budget, sink, recent
    ([1], 16, 1, 1, 0, 0), ([2, 1, 16, 17], 16, 3, 1, 0, 1), ([5], 16, 2, 3, 0, 0),
    ([33, 700, 64], 32, 8, 64, 4, 16), ([1000] * 4, 16, 8, 384, 4, 64),
    ([513, 512, 511], 48, 5, 512, 0, 512), ([4097], 64, 4, 100, 100, 0),
    ([20000, 37], 16, 2, 1024, 4, 128), ([50000], 16, 1, 300, 4, 10), ([3000], 16, 4, 2999, 1, 1),
    ([70000, 300, 9000, 70000], 16, 2, 5000, 20, 333), ([40001] * 3, 48, 3, 39000, 17, 19),
    ([37 * i % 900 + 1 for i in range(40)], 16, 5, 200, 3, 30),
    ([53 * i % 400 + 1 for i in range(130)], 16, 2, 100, 0, 9)]


@pytest.mark.parametrize("case", SELECT)
@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
def test_select(case, kind):
    lens, page, hkv, budget, sink, recent = case
    tables, slots = layout(lens, page, sum(lens))
    rng = np.random.default_rng(len(lens) + budget)
    if kind == "spread":
        x = np.exp(3 * rng.standard_normal((hkv, slots)))
    elif kind == "ties":
        x = rng.integers(0, 3, (hkv, slots)).astype(float)
    else:  # zeros of both signs, infinities, NaN, negative and subnormal numbers
        x = rng.choice([0.0, -0.0, np.inf, -np.inf, np.nan, -1.0, 1e-42, 1.0], (hkv, slots))
    x = x.astype(np.float32)
    want = ref.select(x, tables, lens, page, budget, sink, recent)
    np.testing.assert_array_equal(run_select(x, tables, lens, page, budget, sink, recent), want)


def test_select_longer_than_said():
    """max_len sizes the launch only: longer sequences are read in passes."""
    lens = [900, 40]
    tables, slots = layout(lens, 16, 1)
    x = np.random.default_rng(0).random((2, slots)).astype(np.float32)
    want = ref.select(x, tables, lens, 16, 32, 2, 3)
    for said in (0, 40, 899, 60000):
        np.testing.assert_array_equal(run_select(x, tables, lens, 16, 32, 2, 3, said), want)


def test_select_flags_lists_out_of_range():
    import fekv
    import torch
    from fekv import _lib
    lens = [100, 100, 100]
    tables, slots = layout(lens, 16, 4)
    x = np.random.default_rng(0).random((2, slots)).astype(np.float32)
    want = ref.select(x, tables, lens, 16, 20, 0, 0)
    kv, pages, last = lists(tables, lens, 16)
    for spoil, skipped in ((lambda: last.__setitem__(1, 17), [1]),
                           (lambda: kv.__setitem__(3, 22), [2])):
        spoil()
        kept = torch.zeros(3, 2, 20, dtype=torch.int32, device="cuda")
        fekv.select_tokens(torch.from_numpy(x).cuda(), kv, pages, last, kept, 16, 100)
        assert fekv.device_errors() == _lib.FE_DEVERR_PAGE_RANGE
        full = want.copy()
        full[skipped] = -1
        np.testing.assert_array_equal(kept.cpu().numpy(), full)
        last[1] = (lens[1] - 1) % 16 + 1
    # a page outside the pool: its tokens are the last choice
    kv, pages, last = lists(tables, lens, 16)
    pages[8] = slots // 16  # the second sequence's second page
    y = x.copy()
    y[:, tables[1][1] * 16:tables[1][1] * 16 + 16] = np.nan
    kept = torch.zeros(3, 2, 20, dtype=torch.int32, device="cuda")
    fekv.select_tokens(torch.from_numpy(x).cuda(), kv, pages, last, kept, 16, 100)
    assert fekv.device_errors() == _lib.FE_DEVERR_PAGE_RANGE
    np.testing.assert_array_equal(kept.cpu().numpy(), ref.select(y, tables, lens, 16, 20, 0, 0))


COMPACT = [  # lens, page, hkv, dim, budget, sink, recent
    ([1], 16, 1, 128, 1, 0, 0), ([40, 17, 3], 16, 3, 128, 8, 1, 2), ([575], 16, 8, 128, 512, 4, 64),
    ([700, 33, 64], 32, 4, 256, 64, 4, 16), ([900] * 3, 48, 5, 40, 300, 0, 0),
    ([2000] * 40, 16, 8, 128, 256, 4, 32), ([130], 16, 2, 512, 129, 0, 0)]


def pools(slots, hkv, dim, dtype, seed):
    import torch
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(slots, hkv, dim, generator=gen).to(getattr(torch, dtype))
            for _ in range(2)]


def bits(t):
    import torch
    return t.detach().cpu().contiguous().view(torch.int16).numpy()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("case", COMPACT)
def test_compact_in_place_and_to_other_pages(case, dtype):
    import fekv
    import torch
    lens, page, hkv, dim, budget, sink, recent = case
    tables, slots = layout(lens, page, budget, spare=sum(-(-min(budget, n) // page) for n in lens))
    used = set(np.concatenate(tables).tolist())
    free = [p for p in range(slots // page - 1) if p not in used]
    dst, at = [], 0
    for n in lens:
        need = -(-min(budget, n) // page)
        dst.append(np.array(free[at:at + need]))
        at += need
    rng = np.random.default_rng(1)
    x = rng.random((hkv, slots)).astype(np.float32)
    kept = ref.select(x, tables, lens, page, budget, sink, recent)
    k, v = pools(slots, hkv, dim, dtype, 3)
    for to in (None, dst):
        want_k, want_v, want_x = bits(k).copy(), bits(v).copy(), x.copy()
        ref.compact([want_k, want_v], want_x, kept, tables, lens, page, to)
        kc, vc, xs = k.cuda(), v.cuda(), torch.from_numpy(x).cuda()
        more = {} if to is None else dict(dst_kv=i32(np.cumsum([0] + [len(t) for t in to])),
                                          dst_pages=i32(np.concatenate(to)))
        fekv.compact_tokens(kc, vc, xs, i32(kept), *lists(tables, lens, page), page, **more)
        assert fekv.device_errors() == 0
        np.testing.assert_array_equal(bits(kc), want_k)
        np.testing.assert_array_equal(bits(vc), want_v)
        np.testing.assert_array_equal(xs.cpu().numpy(), want_x)
        # without scores
        kc, vc = k.cuda(), v.cuda()
        fekv.compact_tokens(kc, vc, None, i32(kept), *lists(tables, lens, page), page, **more)
        np.testing.assert_array_equal(bits(kc), want_k)
        np.testing.assert_array_equal(bits(vc), want_v)


def test_compact_skips_and_flags_bad_entries():
    import fekv
    import torch
    from fekv import _lib
    lens, page, hkv, dim = [64, 64], 16, 2, 128
    tables, slots = layout(lens, page, 9)
    kept = np.tile(np.arange(8, 40, 2, dtype=np.int32), (2, 2, 1))
    good = kept.copy()
    kept[0, 1, 3] = 64           # past the sequence
    kept[1, 0, 10] = 2           # before its own place
    k, v = pools(slots, hkv, dim, "bfloat16", 5)
    want_k, want_v = bits(k).copy(), bits(v).copy()
    ref.compact([want_k, want_v], None, good, tables, lens, page)
    for b, h, j in ((0, 1, 3), (1, 0, 10)):  # left as they were
        at = ref.slots_of(tables[b], page, 64)[j]
        want_k[at, h], want_v[at, h] = bits(k)[at, h], bits(v)[at, h]
    kc, vc = k.cuda(), v.cuda()
    fekv.compact_tokens(kc, vc, None, i32(kept), *lists(tables, lens, page), page)
    assert fekv.device_errors() == _lib.FE_DEVERR_PAGE_RANGE
    np.testing.assert_array_equal(bits(kc), want_k)
    np.testing.assert_array_equal(bits(vc), want_v)
    # more tokens than the destination has pages for; a sequence past the lists
    kv, pages, last = lists(tables, lens, page)
    free = [p for p in range(slots // page) if p not in set(np.concatenate(tables).tolist())]
    kc, vc = k.cuda(), v.cuda()
    fekv.compact_tokens(kc, vc, None, i32(good[:, :, :]), kv, pages, last, page,
                        dst_kv=i32([0, 1, 2]), dst_pages=i32(free[:2]))
    assert fekv.device_errors() == 0  # sixteen tokens on one page each
    want_k, want_v = bits(k).copy(), bits(v).copy()
    ref.compact([want_k, want_v], None, good, tables, lens, page, [free[:1], free[1:2]])
    np.testing.assert_array_equal(bits(kc), want_k)
    kc, vc = k.cuda(), v.cuda()
    fekv.compact_tokens(kc, vc, None, i32(good), kv, pages, last, page, dst_kv=i32([0, 0, 1]),
                        dst_pages=i32(free[:1]))
    assert fekv.device_errors() == _lib.FE_DEVERR_PAGE_RANGE
    want_k = bits(k).copy()
    want_v = bits(v).copy()
    none = good.copy()
    none[0] = -1
    ref.compact([want_k, want_v], None, none, tables, lens, page, [free[:1], free[:1]])
    np.testing.assert_array_equal(bits(kc), want_k)
    np.testing.assert_array_equal(bits(vc), want_v)


def test_select_and_compact_replay():
    """Both calls captured in a graph, replayed for later lengths."""
    import fekv
    import torch
    lens, page, hkv, dim, budget = [300, 200, 90], 16, 4, 128, 64
    tables, slots = layout(lens, page, 2)
    kv, pages, last = lists(tables, lens, page)
    x = np.random.default_rng(3).random((hkv, slots)).astype(np.float32)
    k, v = pools(slots, hkv, dim, "float16", 8)
    kc, vc, xs = k.cuda(), v.cuda(), torch.from_numpy(x).cuda()
    kept = torch.zeros(3, hkv, budget, dtype=torch.int32, device="cuda")
    fekv.select_tokens(xs, kv, pages, last, kept, page, 304, sink=2, recent=5)  # warm up
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        fekv.select_tokens(xs, kv, pages, last, kept, page, 304, sink=2, recent=5)
        fekv.compact_tokens(kc, vc, xs, kept, kv, pages, last, page)
    for cut in (0, 3):
        now = [n - cut for n in lens]
        last.copy_(lists(tables, now, page)[2])
        kc.copy_(k)
        vc.copy_(v)
        xs.copy_(torch.from_numpy(x))
        g.replay()
        torch.cuda.synchronize()
        want = ref.select(x, tables, now, page, budget, 2, 5)
        np.testing.assert_array_equal(kept.cpu().numpy(), want)
        want_k, want_v, want_x = bits(k).copy(), bits(v).copy(), x.copy()
        ref.compact([want_k, want_v], want_x, want, tables, now, page)
        np.testing.assert_array_equal(bits(kc), want_k)
        np.testing.assert_array_equal(bits(vc), want_v)
        np.testing.assert_array_equal(xs.cpu().numpy(), want_x)
    assert fekv.device_errors() == 0
