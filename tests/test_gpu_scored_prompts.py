"""Scored attention of whole prompts: more row blocks than a plan's batch and
heads alone would allow, and more records than its first workspace holds."""
import pytest

from test_gpu_scored_attention import check_scores, scored_plan, start
from test_gpu_shared_attention import Step

pytestmark = pytest.mark.gpu


def run(s, plan, graph=False):
    import fekv
    import torch
    plan.prepare(*s.meta(), graph=graph)
    before = start(s)
    out, scores = torch.full_like(s.q, 7.0), before.clone()
    plan.attention(s.q, s.k, s.v, scores, out)
    assert fekv.device_errors() == 0
    s.check(out, True)
    check_scores(s, before, scores, s.rows)


@pytest.mark.parametrize("shape,n", [((128, 8, 128), 1040), ((16, 16, 128), 2100),
                                     ((32, 2, 256), 700)])
def test_prompt_of_one_sequence(shape, n):
    s = Step([(0, [(n, n)])], *shape, 16, "bfloat16")
    run(s, scored_plan(s))


def test_workspace_grows_and_captured_runs_stay():
    """128 heads, 1030 query rows of each of four sequences: 2^26 floats hold the
    records of 4032. A run captured before keeps the workspace that it was
    captured with, lists and records: steps of other workspaces do not reach it."""
    import fekv
    import torch
    big = Step([(0, [(1030, 1030)] * 4)], 128, 8, 128, 16, "bfloat16")
    small = Step([(0, [(300, 4), (77, 4), (20, 4), (500, 4)])], 128, 8, 128, 16, "bfloat16", seed=3)
    slots, n = big.k.shape[0], small.k.shape[0]
    for name in ("k", "v"):  # the same pools for both
        x = torch.zeros_like(getattr(big, name))
        x[:n] = getattr(small, name)
        setattr(small, name, x)
    plan = big.plan(fekv.ScoredPlan, max_keys=4 * 1030 * 1040)
    plan.prepare(*small.meta(), graph=True)
    before = start(small)
    out, scores = torch.zeros_like(small.q), before.clone()
    plan.attention(small.q, small.k, small.v, scores, out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan.attention(small.q, small.k, small.v, scores, out)
    run(big, plan)
    assert plan.info()["partial_floats"] > 1 << 26
    for again in (False, True, True):
        if again:
            plan.prepare(*small.meta(), graph=True)
        scores.copy_(before)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        small.check(out, True)
        check_scores(small, before, scores, small.rows)
        run(big, plan)
    assert slots == small.k.shape[0] and fekv.device_errors() == 0


def test_graph_of_many_rows():
    """A graph prepare sizes the workspace for later steps of as many rows, cut in
    other places."""
    import fekv
    import torch
    steps = [Step([(0, [(n, 1030) for n in lens])], 128, 8, 128, 16, "bfloat16", seed=len(lens))
             for lens in ((1030, 1060, 1090, 1120), (1100, 1030, 1300, 1033))]
    slots = max(s.k.shape[0] for s in steps)
    plan = fekv.ScoredPlan(128, 8, 128, 16, 4, 90, True, slots // 16 - 1, max_keys=5 * 1030 * 1328)
    k, v = (torch.zeros(slots, 8, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    q, out = torch.zeros_like(steps[0].q), torch.zeros_like(steps[0].q)
    scores = torch.zeros(8, slots, device="cuda")
    plan.prepare(*steps[0].meta(), graph=True)
    plan.attention(q, k, v, scores, out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan.attention(q, k, v, scores, out)
    for s in steps[::-1] + steps:
        n = s.k.shape[0]
        k[:n].copy_(s.k)
        v[:n].copy_(s.v)
        q.copy_(s.q)
        before = start(s)
        scores[:, :n].copy_(before)
        plan.prepare(*s.meta(), graph=True)
        g.replay()
        torch.cuda.synchronize()
        s.check(out, True)
        check_scores(s, before, scores[:, :n], s.rows)
    assert fekv.device_errors() == 0
