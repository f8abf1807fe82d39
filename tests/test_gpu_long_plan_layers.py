"""A plan for long shared prompts over the pools of a model's layers: one prepare,
a run per layer, eager and captured."""
import pytest

import long_ref as ref
from test_gpu_scored_attention import check_scores, start
from test_gpu_shared_attention import Step, ones

pytestmark = pytest.mark.gpu

LAYERS = 3


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("scored", [False, True])
@pytest.mark.parametrize("shape", [(32, 8, 128), (16, 2, 256), (5, 5, 256)])
def test_layers_in_turn(shape, scored, captured):
    import fekv
    import torch
    layout = [(0, ones(5, 33, 700) + [(90, 7)])] if scored else [(24, ones(*range(1, 41))),
                                                               (0, [(200, 40)])]
    s = Step(layout, *shape, 16, "bfloat16")
    used = [ref.slots_of(t, 16, n) for t, n in zip(s.tables, s.lens)]
    pools = [(s.k, s.v)] + [ref.pools(s.blocks, 16, *shape[1:], s.dtype, used, 50 + i)
                            for i in range(LAYERS - 1)]
    gen = torch.Generator(device="cuda").manual_seed(9)
    qs = [torch.randn(s.q.shape, generator=gen, device="cuda").to(s.dtype) for _ in pools]
    befores = [start(s, 70 + i) for i in range(LAYERS)]
    outs = [torch.zeros_like(s.q) for _ in pools]
    scores = [b.clone() for b in befores]
    plan = s.plan(fekv.ScoredPlan, max_keys=4000) if scored else s.plan()
    plan.prepare(*s.meta(), graph=captured)

    def layers():
        for q, (k, v), x, o in zip(qs, pools, scores, outs):
            if scored:
                plan.attention(q, k, v, x, o)
            else:
                plan.attention(q, k, v, o)

    layers()
    if captured:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            layers()
        for x, b, o in zip(scores, befores, outs):
            x.copy_(b)
            o.zero_()
        g.replay()
        torch.cuda.synchronize()
    assert fekv.device_errors() == 0
    for q, (k, v), x, b, o in zip(qs, pools, scores, befores, outs):
        s.q, s.k, s.v = q, k, v
        s.check(o, True)
        if scored:
            check_scores(s, b, x, s.rows)
