"""Attention that scores the keys against the definition in 64 bits, and the
way of a prompt through score, selection and compaction."""
import numpy as np
import pytest

import evict_ref
import long_ref as ref
from test_gpu_shared_attention import Step, ones

pytestmark = pytest.mark.gpu


def scored_plan(s):
    import fekv
    return s.plan(fekv.ScoredPlan,
                  max_keys=sum(r * (n + 15) for n, r in zip(s.lens, s.rows)))


def start(s, seed=3):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.rand(s.hkv, s.k.shape[0], generator=gen, device="cuda") * 4


def check_scores(s, before, after, fresh):
    import torch
    want, limit = before.double(), torch.zeros_like(before, dtype=torch.float64)
    at = 0
    for t, n, r, f in zip(s.tables, s.lens, s.rows, fresh):
        if r == 0:
            continue
        slots = torch.from_numpy(ref.slots_of(t, s.page, n)).cuda()
        w, bound = ref.attend(s.q[at:at + r], s.k[slots], s.v[slots], True)[2:]
        want[:, slots[n - f:]] = 0
        want[:, slots] += w
        limit[:, slots] = bound
        at += r
    # one rounding of the sum, and each weight's own
    off = (after.double() - want).abs()
    assert ((off - limit - 2.0 ** -23 * want.abs()) <= 0).all(), (off - limit).max()


LAYOUTS = {
    "few": ones(1, 5, 33, 700),
    "many": ones(*range(1, 61)),
    "drafts": [(4, 4), (200, 3), (37, 0), (16, 16), (5, 5), (1000, 2)],
    "window": [(900, 32), (33, 33), (515, 40)],
}
SHAPES = [(16, 8, 128, 16), (32, 4, 128, 16), (40, 8, 128, 32), (6, 3, 128, 48), (16, 1, 128, 16),
          (16, 2, 256, 16), (5, 5, 256, 64), (8, 8, 128, 16), (12, 4, 128, 16)]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("name", LAYOUTS)
def test_against_64_bits(name, shape, dtype):
    import fekv
    import torch
    s = Step([(0, LAYOUTS[name])], *shape[:3], shape[3], dtype, seed=len(name))
    plan = scored_plan(s)
    before = start(s)
    for fresh in (None, [0] * len(s.lens), [n - n // 3 for n in s.lens], s.lens):
        plan.prepare(*s.meta(), fresh=fresh)
        out, scores = torch.full_like(s.q, 7.0), before.clone()
        plan.attention(s.q, s.k, s.v, scores, out)
        assert fekv.device_errors() == 0
        s.check(out, True)
        check_scores(s, before, scores, s.rows if fresh is None else fresh)
    again, scores2 = torch.empty_like(s.q), before.clone()
    plan.attention(s.q, s.k, s.v, scores2, again)
    assert torch.equal(out, again) and torch.equal(scores, scores2)


def test_long_context_of_one_sequence():
    import torch
    s = Step([(0, ones(20001))], 8, 2, 128, 16, "bfloat16")
    plan = scored_plan(s)
    plan.prepare(*s.meta())
    before = start(s)
    out, scores = torch.empty_like(s.q), before.clone()
    plan.attention(s.q, s.k, s.v, scores, out)
    s.check(out, True)
    check_scores(s, before, scores, [1])


def test_weights_of_a_row_add_up_to_one():
    """Set and not added to, the scores of a sequence sum to its query rows
    times the heads of each KV head: to n 2^-20 of it for n = 1000 keys' sums."""
    import torch
    s = Step([(0, [(1000, 6)])], 12, 4, 128, 16, "float16")
    plan = scored_plan(s)
    plan.prepare(*s.meta(), fresh=s.lens)
    scores = start(s)
    plan.attention(s.q, s.k, s.v, scores, torch.empty_like(s.q))
    got = scores[:, torch.from_numpy(ref.slots_of(s.tables[0], 16, 1000)).cuda()].double().sum(1)
    assert (got - 18).abs().max() < 18 * 2e-3  # d of long_ref for these sizes is 1e-3


def test_replay_for_other_lengths():
    import fekv
    import torch
    layouts = [ones(*range(1, 25)), ones(*[400] * 24), ones(*[16] * 23, 3000)]
    steps = [Step([(0, g)], 32, 8, 128, 16, "bfloat16", seed=i) for i, g in enumerate(layouts)]
    slots = max(s.k.shape[0] for s in steps)
    plan = fekv.ScoredPlan(32, 8, 128, 16, 24, 200, True, slots // 16 - 1, max_keys=24 * 416)
    k, v = (torch.zeros(slots, 8, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q, out = torch.zeros_like(steps[0].q), torch.zeros_like(steps[0].q)
    scores = torch.zeros(8, slots, device="cuda")
    plan.prepare(*steps[0].meta(), graph=True)
    plan.attention(q, k, v, scores, out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan.attention(q, k, v, scores, out)
    for s in steps + steps[:1]:
        n = s.k.shape[0]
        k[:n].copy_(s.k)
        v[:n].copy_(s.v)
        q.copy_(s.q)
        before = start(s)
        scores.zero_()
        scores[:, :n].copy_(before)
        plan.prepare(*s.meta(), graph=True)
        g.replay()
        torch.cuda.synchronize()
        s.check(out, True)
        check_scores(s, before, scores[:, :n], s.rows)
        assert not scores[:, n:].any()
    assert fekv.device_errors() == 0


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_prompt_scored_selected_compacted_and_continued(dtype):
    """The whole way: keys rotated at three axes into the cache, the prompt's last rows
    scored, each KV head cut to its best keys, and a decode step over what is
    left, against attention over the kept keys of each head in 64 bits."""
    import fekv
    import torch
    from test_gpu_rope_axes import rotated
    hq, hkv, dim, page, budget, sink, recent, window = 16, 8, 128, 16, 96, 4, 24, 16
    lens = [300, 64, 411]
    rng = np.random.default_rng(4)
    _, tables, blocks = ref.tables([n + 1 for n in lens], page, 5)
    dt = getattr(torch, dtype)
    slots = (blocks + 1) * page
    kc, vc = (torch.full((slots, hkv, dim), float("nan"), dtype=dt, device="cuda")
              for _ in range(2))
    pairs = fekv.rope_sections((24, 20, 20), True)
    ang = rng.uniform(0, 7, (512, dim // 2))
    cache = np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32)
    cache_d = torch.from_numpy(cache).cuda()

    def append(rows, at, pos):
        """New rows at the slots `at`: their rotated queries."""
        q, k, v = (torch.from_numpy(rng.standard_normal((rows, h, dim)).astype(np.float32)).to(dt)
                   for h in (hq, hkv, hkv))
        d = [x.cuda() for x in (q, k, v)]
        fekv.rope_axes_append(*d, kc, vc, torch.from_numpy(at).cuda(),
                              torch.from_numpy(pos).cuda(), cache_d, pairs)
        want = torch.from_numpy(rotated(k.float().numpy(), pos, cache, pairs)).to(dt)
        assert torch.equal(kc[torch.from_numpy(at).cuda()].cpu(), want)
        return d[0]

    i32 = lambda v: torch.tensor(np.asarray(v, np.int32), device="cuda")  # noqa: E731
    cum = lambda v: np.cumsum([0] + list(v)).astype(np.int32)  # noqa: E731
    at = [ref.slots_of(t, page, n) for t, n in zip(tables, lens)]
    q = append(sum(lens), np.concatenate(at), rng.integers(0, 512, (3, sum(lens))))
    ends = np.cumsum(lens)
    q = torch.cat([q[e - window:e] for e in ends]).contiguous()
    scores = torch.full((hkv, slots), 1e9, device="cuda")  # stale: every key is fresh
    plan = fekv.ScoredPlan(hq, hkv, dim, page, 3, max(map(len, tables)), dtype == "bfloat16",
                           blocks, max_keys=sum((n + 16) * window for n in lens))
    pages = np.concatenate(tables)
    kv = cum(len(t) for t in tables)
    cut = [t[:-(-n // page)] for t, n in zip(tables, lens)]
    last = [(n - 1) % page + 1 for n in lens]
    plan.prepare(cum([window] * 3), cum(map(len, cut)), np.concatenate(cut), last, fresh=lens)
    plan.attention(q, kc, vc, scores, torch.empty_like(q))
    kept = torch.empty(3, hkv, budget, dtype=torch.int32, device="cuda")
    lists = (i32(cum(map(len, cut))), i32(np.concatenate(cut)), i32(last))
    fekv.select_tokens(scores, *lists, kept, page, max(lens), sink=sink, recent=recent)
    want = evict_ref.select(scores.cpu().numpy(), cut, lens, page, budget, sink, recent)
    np.testing.assert_array_equal(kept.cpu().numpy(), want)
    k0, v0, x0 = kc.clone(), vc.clone(), scores.clone()
    fekv.compact_tokens(kc, vc, scores, kept, *lists, page)
    left = [min(n, budget) for n in lens]
    # one token more for each: appended behind the kept ones, then attended
    new = np.array([ref.slots_of(t, page, n + 1)[n] for t, n in zip(tables, left)])
    q = append(3, new, rng.integers(0, 512, (3, 3)))
    tabs = [t[:-(-(n + 1) // page)] for t, n in zip(tables, left)]
    plan.prepare(cum([1] * 3), cum(map(len, tabs)), np.concatenate(tabs),
                 [n % page + 1 for n in left])
    out = torch.empty_like(q)
    before = scores.clone()
    plan.attention(q, kc, vc, scores, out)
    G = hq // hkv
    for b, n in enumerate(left):
        src = torch.from_numpy(at[b]).cuda()
        for h in range(hkv):
            pick = src[torch.from_numpy(want[b, h, :n].astype(np.int64)).cuda()]
            k = torch.cat([k0[pick, h], kc[new[b], h][None]])[:, None]
            v = torch.cat([v0[pick, h], vc[new[b], h][None]])[:, None]
            o, bound, w, wb = ref.attend(q[b:b + 1, h * G:h * G + G], k, v, True)
            ref.check_output(out[b:b + 1, h * G:h * G + G], o, bound)
            dst = torch.from_numpy(ref.slots_of(tables[b], page, n + 1)).cuda()
            old = torch.cat([x0[h, pick], torch.zeros(1, device="cuda")]).double()
            off = (scores[h, dst].double() - old - w[0]).abs()
            assert (off <= wb[0] + 2.0 ** -23 * (old + w[0])).all()
            assert torch.equal(before[h, dst[:n]], x0[h, pick])
    assert fekv.device_errors() == 0
    assert len(pages) == kv[-1]
