"""Lists of kept tokens that other callers than select_tokens write: a list ends at
its first -1, whatever stands behind."""
import numpy as np
import pytest

import evict_ref as ref
from test_gpu_evict import bits, i32, layout, lists, pools

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("to_others", [False, True])
@pytest.mark.parametrize("end", [0, 1, 37, 255, 256, 257, 300, 511, 512, 599, 600])
def test_a_list_ends_at_its_first_minus_one(end, to_others):
    """The entries behind it name tokens of the sequence, tokens far past it and
    more -1: none is moved, none is flagged."""
    import fekv
    import torch
    page, hkv, dim, budget = 16, 3, 128, 600
    n = [1300, 1250]
    tables, slots = layout(n, page, end, spare=80)
    used = set(np.concatenate(tables).tolist())
    free = [p for p in range(slots // page - 1) if p not in used]
    dst = [np.array(free[:38]), np.array(free[38:76])] if to_others else None
    rng = np.random.default_rng(end)
    kept = np.stack([[np.sort(rng.choice(1200, budget, replace=False)) for _ in range(hkv)]
                     for _ in n]).astype(np.int32)
    kept[:, :, end:end + 1] = -1
    behind = kept[:, :, end + 1:]
    behind[:, :, 1::3] = -1
    behind[:, 1, 2::3] = 1 << 30  # past the sequence
    kept[1, 2] = np.arange(100, 700)  # and a list that is whole
    k, v = pools(slots, hkv, dim, "bfloat16", 7)
    x = rng.random((hkv, slots)).astype(np.float32)
    want_k, want_v, want_x = bits(k).copy(), bits(v).copy(), x.copy()
    ref.compact([want_k, want_v], want_x, kept, tables, n, page, dst)
    kc, vc, xs = k.cuda(), v.cuda(), torch.from_numpy(x).cuda()
    more = {} if dst is None else dict(dst_kv=i32([0, 38, 76]), dst_pages=i32(np.concatenate(dst)))
    fekv.compact_tokens(kc, vc, xs, i32(kept), *lists(tables, n, page), page, **more)
    assert fekv.device_errors() == 0
    np.testing.assert_array_equal(bits(kc), want_k)
    np.testing.assert_array_equal(bits(vc), want_v)
    np.testing.assert_array_equal(xs.cpu().numpy(), want_x)


def test_a_bad_entry_before_the_end_is_flagged():
    import fekv
    from fekv import _lib
    page, hkv, dim = 16, 2, 128
    tables, slots = layout([400], page, 3)
    kept = np.full((1, hkv, 350), -1, np.int32)
    kept[:, :, :300] = np.arange(50, 350)
    k, v = pools(slots, hkv, dim, "float16", 7)
    for at, what in ((299, 400), (10, 5), (300, 7)):  # past the sequence, before its own place
        bad = kept.copy()
        bad[0, 1, at] = what
        if at == 300:
            bad[0, 1, 300:302] = -1, what  # behind the end
        kc, vc = k.cuda(), v.cuda()
        fekv.compact_tokens(kc, vc, None, i32(bad), *lists(tables, [400], page), page)
        assert fekv.device_errors() == (0 if at == 300 else _lib.FE_DEVERR_PAGE_RANGE)
