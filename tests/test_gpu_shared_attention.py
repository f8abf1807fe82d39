"""Attention over shared prefixes against the definition in 64 bits (long_ref:
the bound of every rounding), with pools that hold NaN in every slot that no
sequence uses."""
import numpy as np
import pytest

import long_ref as ref

pytestmark = pytest.mark.gpu


class Step:
    """groups: (prefix pages, [(own tokens, query rows), ...]) each."""

    def __init__(self, groups, hq, hkv, dim, page, dtype, seed=0, slack=0):
        import torch
        self.hq, self.hkv, self.dim, self.page = hq, hkv, dim, page
        self.dtype = getattr(torch, dtype)
        own = [n for _, m in groups for n, _ in m]
        heads, tabs, self.blocks = ref.tables(own, page, seed, [p for p, _ in groups])
        self.tables, self.lens, self.rows = [], [], []
        for g, (p, members) in enumerate(groups):
            for n, r in members:
                self.tables.append(np.concatenate([heads[g], tabs[len(self.tables)]]))
                self.lens.append(p * page + n)
                self.rows.append(r)
        used = [ref.slots_of(t, page, n) for t, n in zip(self.tables, self.lens)]
        self.k, self.v = ref.pools(self.blocks, page, hkv, dim, self.dtype, used, seed)
        gen = torch.Generator(device="cuda").manual_seed(seed + 1)
        self.q = (torch.randn(sum(self.rows) + slack, hq, dim, generator=gen, device="cuda") *
                  1.5).to(self.dtype)

    def meta(self):
        cum = lambda v: np.cumsum([0] + list(v)).astype(np.int32)  # noqa: E731
        return (cum(self.rows), cum(len(t) for t in self.tables), np.concatenate(self.tables),
                np.array([(n - 1) % self.page + 1 for n in self.lens], np.int32))

    def plan(self, kind=None, **more):
        import fekv
        return (kind or fekv.SharedPlan)(self.hq, self.hkv, self.dim, self.page, len(self.tables),
                                         max(map(len, self.tables)), self.q.dtype.itemsize == 2 and
                                         "bfloat" in str(self.dtype), self.blocks, **more)

    def check(self, out, causal):
        import torch
        at = 0
        for t, n, r in zip(self.tables, self.lens, self.rows):
            slots = torch.from_numpy(ref.slots_of(t, self.page, n)).cuda()
            if r:
                want, bound = ref.attend(self.q[at:at + r], self.k[slots], self.v[slots],
                                         causal)[:2]
                ref.check_output(out[at:at + r], want, bound)
            at += r


def ones(*lens):
    return [(n, 1) for n in lens]


LAYOUTS = {
    # one group whose rows fit the decode kernel's block, and one that is no group
    "few": [(32, ones(1, 5, 33)), (0, ones(70))],
    # many single rows: the prefix runs on the row kernel
    "many": [(24, ones(*range(1, 61)))],
    # three prefixes, the last too short to be worth sharing
    "three": [(20, ones(*[7] * 40)), (40, ones(*range(3, 40))), (1, ones(2, 9))],
    # draft blocks of several rows, some of them long; one member without rows
    "drafts": [(30, [(4, 4)] * 9 + [(20, 3), (3, 0), (16, 16)] + [(5, 5)] * 8)],
    # verification blocks: items of one and of two row tiles, of one and of several
    # key tiles, one behind the other on an SM
    "blocks": [(70, [(16 + 23 * i % 300, 16) for i in range(40)]),
               (0, [(200, 40), (333, 9), (90, 20), (17, 17)]),
               (33, [(64 + i, 33) for i in range(0, 300, 17)])],
    # a prefill chunk over the prefix beside decode rows
    "chunk": [(26, [(300, 300)] + ones(*range(1, 30)))],
}
SHAPES = [(16, 8, 128, 16), (32, 4, 128, 16), (40, 8, 128, 32), (6, 3, 128, 48), (16, 1, 128, 16),
          (16, 2, 256, 16), (5, 5, 256, 64), (8, 8, 128, 16)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("name", LAYOUTS)
def test_against_64_bits(name, shape, dtype, causal):
    import fekv
    import torch
    s = Step(LAYOUTS[name], *shape[:3], shape[3], dtype, seed=len(name) + shape[0])
    plan = s.plan()
    plan.prepare(*s.meta())
    out = torch.full_like(s.q, 7.0)
    plan.attention(s.q, s.k, s.v, out, causal)
    assert fekv.device_errors() == 0
    s.check(out, causal)
    again = torch.empty_like(s.q)
    plan.attention(s.q, s.k, s.v, again, causal)
    assert torch.equal(out, again)  # no order of arrival in the sums


def test_what_is_shared():
    """Groups are found, and taken where they pay."""
    s = Step(LAYOUTS["three"], 32, 8, 128, 16, "bfloat16")
    plan = s.plan()
    plan.prepare(*s.meta())
    assert plan.info()["shared_groups"] == 2
    plan.prepare(*s.meta(), groups=([0, len(s.tables)], [0]))
    assert plan.info()["shared_groups"] == 0


@pytest.mark.parametrize("causal", [True, False])
def test_shared_pages_that_reach_query_rows(causal):
    """All pages of the members are the same (samples of one prompt): the
    pages that hold query rows are read by each."""
    import torch
    s = Step([(40, [(1, 1)])], 16, 8, 128, 16, "float16")
    n = 12
    s.tables, s.lens, s.rows = s.tables * n, [41 * 16 - 15] * n, [1] * n
    s.rows[3] = 20  # its first rows lie on the prefix's last page
    gen = torch.Generator(device="cuda").manual_seed(5)
    s.q = torch.randn(sum(s.rows), 16, 128, generator=gen, device="cuda").to(s.dtype)
    plan = s.plan()
    plan.prepare(*s.meta(), groups=([0, n], [41]))
    assert plan.info()["shared_groups"] == 1
    out = torch.empty_like(s.q)
    plan.attention(s.q, s.k, s.v, out, causal)
    s.check(out, causal)


def test_long_prefix_and_many_pieces():
    """One short group over a long prefix: pieces of it on every SM, joined
    from more than 32 records."""
    import torch
    s = Step([(1250, ones(1, 40))], 4, 1, 128, 16, "bfloat16")
    plan = s.plan()
    plan.prepare(*s.meta())
    assert plan.info()["shared_groups"] == 1
    out = torch.empty_like(s.q)
    plan.attention(s.q, s.k, s.v, out)
    s.check(out, True)


def test_one_sequence_and_one_key():
    import torch
    for lens in ([1], [16], [17]):
        s = Step([(0, ones(*lens))], 16, 2, 256, 16, "bfloat16")
        plan = s.plan()
        plan.prepare(*s.meta())
        out = torch.empty_like(s.q)
        plan.attention(s.q, s.k, s.v, out)
        s.check(out, True)


def test_rows_past_the_step_stay():
    import torch
    s = Step(LAYOUTS["many"], 32, 8, 128, 16, "float16", slack=5)
    plan = s.plan()
    plan.prepare(*s.meta())
    out = torch.full_like(s.q, 3.0)
    plan.attention(s.q, s.k, s.v, out)
    assert (out[-5:] == 3.0).all()
    s.check(out, True)


def test_replay_for_other_lengths_and_groups():
    """A captured run serves later prepares: other lengths, other prefixes,
    none, and the decode kernel's share instead of the row kernel's."""
    import torch
    layouts = [[(24, ones(*range(1, 41)))], [(0, ones(*[200] * 40))],
               [(60, ones(*[9] * 17)), (3, ones(*[20] * 23))], [(18, ones(4, 5)),
                                                                (25, ones(*[8] * 38))]]
    steps = [Step(g, 32, 8, 128, 16, "bfloat16", seed=i) for i, g in enumerate(layouts)]
    slots = max(s.k.shape[0] for s in steps)
    blocks = slots // 16 - 1
    import fekv
    plan = fekv.SharedPlan(32, 8, 128, 16, 40, 128, True, blocks)
    k, v = (torch.zeros(slots, 8, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q, out = torch.zeros_like(steps[0].q), torch.zeros_like(steps[0].q)
    plan.prepare(*steps[0].meta(), graph=True)
    plan.attention(q, k, v, out)  # loads the kernels
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan.attention(q, k, v, out)
    for s in steps + steps[:1]:
        k[:s.k.shape[0]].copy_(s.k)
        v[:s.v.shape[0]].copy_(s.v)
        q.copy_(s.q)
        plan.prepare(*s.meta(), graph=True)
        g.replay()
        torch.cuda.synchronize()
        s.check(out, True)
    assert fekv.device_errors() == 0


def test_on_another_stream():
    import torch
    s = Step(LAYOUTS["many"], 16, 8, 128, 16, "bfloat16")
    plan = s.plan()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    out = torch.zeros_like(s.q)
    torch.cuda.synchronize()
    plan.prepare(*s.meta(), stream=side)
    plan.attention(s.q, s.k, s.v, out, stream=side)
    side.synchronize()
    s.check(out, True)
